"""The entries for several requests (xjh_page_plan, xjh_paged_store, xjh_attn_paged, xjh_attn_packed) against plain
forms written here from the text of xj_hip.h, and what they refuse (on the CPU, where nothing is launched).

Tables, lengths and slots are whole numbers and equal. A stored element is its row's, rounded once to nearest: equal bits.
"""
import ctypes as C

import numpy as np
import pytest

import xjpipe as xp


# ------------------------------------------------------------ plain forms --

def bf16_bits(x):
    """float32 to bf16 bits, to nearest, ties to even; NaN stays one."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def up(n, page):
    return -(-n // page)


class RefPool:
    """xjh_page_plan request by request, in Python lists."""

    def __init__(self, page, n_pages, n_req, max_blocks):
        self.page, self.n_pages, self.L = page, n_pages, max_blocks * page
        self.table, self.free = [[-1] * max_blocks for _ in range(n_req)], list(range(n_pages))

    def plan(self, n_past, n_new, held=None, T=None):
        P, L = self.page, self.L
        past, new = [min(max(n, 0), L) for n in n_past], [max(n, 0) for n in n_new]
        held = past if held is None else [min(max(n, 0), L) for n in held]
        kv = [min(p + n, L) for p, n in zip(past, new)]
        for row, h, n in zip(self.table, held, kv):
            self.free += row[up(n, P):up(h, P)]
        want = sum(max(0, up(n, P) - up(h, P)) for h, n in zip(held, kv))
        missing = max(0, want - len(self.free))
        pos, slot, cu = [], [], [0]
        for row, h, p, m, n in zip(self.table, held, past, new, kv):
            for b in range(up(h, P), up(n, P)):
                row[b] = -1 if missing else self.free.pop()
            pos += range(p, p + m)
            slot += [row[q // P] * P + q % P if q < L and row[q // P] >= 0 else -1 for q in range(p, p + m)]
            cu.append(cu[-1] + m)
        T = cu[-1] if T is None else T
        pad = max(0, T - cu[-1])
        return {"cu": cu, "kv_len": kv, "pos": (pos + [0] * pad)[:T], "slot": (slot + [-1] * pad)[:T],
                "status": [missing, sum(max(0, p + m - L) for p, m in zip(past, new)), max(0, cu[-1] - T), cu[-1]]}


def same_plan(pool, ref, **step):
    got, want = pool.plan(**step), ref.plan(**step)
    for k in want:
        assert got[k].tolist() == want[k], k
    assert pool.table.tolist() == ref.table
    assert pool.free.tolist() == ref.free
    return got


# ------------------------------------------------------------------- plan --

@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_plan_steps_of_a_batch(page):
    """Prompts, single tokens, drafts given up, requests that end and begin anew."""
    n_req, blocks = 7, 9
    pool, ref = xp.PagePool(page, 40, n_req, blocks), RefPool(page, 40, n_req, blocks)
    rng = np.random.default_rng(page)
    past = np.zeros(n_req, int)
    new = rng.integers(0, 2 * page + 3, n_req)
    same_plan(pool, ref, n_past=past.tolist(), n_new=new.tolist())
    for step in range(12):
        held = past + new
        keep = held - rng.integers(0, 6, n_req) * (rng.random(n_req) < 0.4)   # rejected drafts
        keep[rng.random(n_req) < 0.15] = 0                                    # over
        past = np.maximum(keep, 0)
        new = np.where(past == 0, rng.integers(0, page + 2, n_req), rng.integers(0, 7, n_req))
        new = np.minimum(new, blocks * page - past)
        got = same_plan(pool, ref, n_past=past.tolist(), n_new=new.tolist(), held=held.tolist(), T=int(new.sum()) + step % 3)
        assert got["status"][0] == 0
        live = [p for row, n in zip(pool.table.tolist(), got["kv_len"]) for p in row[:up(int(n), page)]]
        assert sorted(live + pool.free.tolist()) == list(range(40))   # every page has one owner


@pytest.mark.gpu
def test_plan_edges():
    # no request; no token; no page needed
    pool, ref = xp.PagePool(16, 3, 0, 1), RefPool(16, 3, 0, 1)
    assert same_plan(pool, ref, n_past=[], n_new=[], T=2)["slot"].tolist() == [-1, -1]
    pool, ref = xp.PagePool(16, 3, 2, 4), RefPool(16, 3, 2, 4)
    same_plan(pool, ref, n_past=[0, 0], n_new=[0, 0])
    # negative lengths, and lengths beyond the row
    same_plan(pool, ref, n_past=[-5, 0], n_new=[-1, 17])
    # a step that lacks a page takes none, and can be tried again with less
    got = same_plan(pool, ref, n_past=[0, 17], n_new=[17, 0], T=17)
    assert got["status"].tolist() == [1, 0, 0, 17] and set(got["slot"]) == {-1} and pool.free.size == 1
    got = same_plan(pool, ref, n_past=[0, 17], n_new=[16, 0])
    assert got["status"][0] == 0 and pool.free.size == 0
    # rows beyond T are counted and not written; beyond the table's rows there are no slots
    got = same_plan(pool, ref, n_past=[0, 0], n_new=[0, 0], held=[16, 17])
    got = same_plan(pool, ref, n_past=[0, 0], n_new=[5, 3], T=6)
    assert got["status"].tolist() == [0, 0, 2, 8]
    pool, ref = xp.PagePool(16, 9, 2, 2), RefPool(16, 9, 2, 2)
    got = same_plan(pool, ref, n_past=[30, 500], n_new=[5, 1], held=[0, 0])
    assert got["status"].tolist() == [0, 4, 0, 6] and got["kv_len"].tolist() == [32, 32]


@pytest.mark.gpu
@pytest.mark.parametrize("n_req", [1, 63, 64, 65, 1023, 1024, 1025, 5000])
def test_plan_many_requests(n_req):
    rng = np.random.default_rng(n_req)
    new = rng.integers(0, 40, n_req)
    pages = int(sum(up(int(n), 16) for n in new)) + n_req
    pool, ref = xp.PagePool(16, pages, n_req, 4), RefPool(16, pages, n_req, 4)
    same_plan(pool, ref, n_past=[0] * n_req, n_new=new.tolist())
    past = np.where(rng.random(n_req) < 0.3, 0, new)
    same_plan(pool, ref, n_past=past.tolist(), n_new=[1] * n_req, held=new.tolist())


def test_plan_refusals():
    L, err, one = xp.lib(), C.create_string_buffer(512), C.c_void_p(16)

    def plan(page=16, n_pages=4, blocks=2, n_req=1, T=1, table=16, free=16, n_free=one, out=one, cu=one, kv=one, past=one, new=one,
             status=one, work=one, wb=1 << 20):
        p = xp.XjhPages(page, n_pages, blocks, table, free)
        return L.xjh_page_plan(C.byref(p), None, past, new, n_req, n_free, out, T, cu, kv, None, None, status, work, wb, None, err, 512)

    for bad in ({"page": 8}, {"page": 48}, {"page": 512}, {"n_pages": 0}, {"n_pages": 1 << 27}, {"blocks": 0}, {"blocks": 1 << 27},
                {"n_req": -1}, {"n_req": 65537}, {"n_req": 65536, "blocks": 1 << 15}, {"T": -1}):
        assert plan(**bad) == -1 and b"bad shape" in err.value, bad
    for bad in ({"table": None}, {"free": None}, {"n_free": None}, {"out": None}, {"cu": None}, {"kv": None}, {"past": None}, {"new": None},
                {"status": None}):
        assert plan(**bad) == -1 and b"a buffer is missing" in err.value, bad
    for bad in ({"work": None}, {"work": C.c_void_p(24)}, {"wb": L.xjh_page_plan_work_bytes(1) - 1}):
        assert plan(**bad) == -1 and b"work area" in err.value, bad
    assert L.xjh_page_plan(None, None, one, one, 1, one, one, 1, one, one, None, None, one, one, 1 << 20, None, err, 512) == -1
    assert L.xjh_page_plan_work_bytes(-1) == 0 and L.xjh_page_plan_work_bytes(65537) == 0
    for bad in ((16, 0, 1, 1), (16, 4, 1, 0), (16, 1 << 27, 1, 1), (16, 4, -1, 1), (1 << 31, 4, 1, 1)):
        with pytest.raises(xp.XjError):
            xp.PagePool(*bad)


# ------------------------------------------------------------------ store --

@pytest.mark.gpu
@pytest.mark.parametrize("rows,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("Hkv,D,page,T", [(1, 64, 16, 1), (3, 128, 32, 45), (4, 256, 64, 130), (2, 64, 256, 300)])
def test_store(rows, cache, Hkv, D, page, T):
    rng = np.random.default_rng(T)
    n_pages = up(T, page) + 2
    kv = xp.PagedKv(Hkv, D, page, n_pages, type=xp.F16 if cache == "f16" else xp.BF16)
    before = [rng.integers(0, 0x7000, kv.c.bytes // 2).astype(np.uint16) for _ in range(2)]
    kv.k.put(before[0]), kv.v.put(before[1])
    k, v = ((rng.standard_normal((T, Hkv, D)) * 10.0 ** rng.integers(-9, 6, (T, 1, 1))).astype(np.float32) for _ in range(2))
    k.flat[:min(8, k.size)] = [np.inf, -np.inf, np.nan, 65519.9, 65520.0, -0.0, 1e-30, 2.0 ** -25][:min(8, k.size)]
    slot = rng.permutation(n_pages * page)[:T]
    slot[rng.random(T) < 0.1] = -1
    slot[T // 2] = [-1 << 31, n_pages * page, (1 << 31) - 1][T % 3]
    to = {"f32": lambda x: x, "f16": lambda x: x.astype(np.float16), "bf16": bf16_bits}
    as_cache = {"f16": lambda x: x.astype(np.float16).view(np.uint16), "bf16": bf16_bits}
    with np.errstate(over="ignore"):
        kv.store(to[rows](k), to[rows](v), slot)
        for x, old, got in zip((k, v), before, kv.pages()):
            want = old.reshape(n_pages, Hkv, page, D).copy()
            for t, s in enumerate(slot):
                if 0 <= s < n_pages * page:
                    want[s // page, :, s % page] = as_cache[cache](x[t])
            got = got.view(np.uint16)
            nan = {"f16": lambda b: (b & 0x7FFF) > 0x7C00, "bf16": lambda b: (b & 0x7FFF) > 0x7F80}[cache]
            assert np.array_equal(nan(got), nan(want)) and np.array_equal(np.where(nan(got), 0, got), np.where(nan(want), 0, want))


@pytest.mark.gpu
def test_store_of_strided_unaligned_rows():
    """Rows that begin at any element and lie apart."""
    rng, err = np.random.default_rng(5), C.create_string_buffer(512)
    for dt, t, shift, tok in ((np.float32, xp.F32, 1, 131), (np.float32, xp.F32, 3, 128), (np.float16, xp.F16, 1, 129), (np.float16, xp.F16, 5, 200)):
        kv = xp.PagedKv(2, 64, 16, 2)
        T, buf = 9, rng.standard_normal(2000).astype(dt)
        d, slot = xp.Dev(buf), xp.Dev(np.arange(T, dtype=np.int32) * 3)
        at = d.ptr + shift * buf.itemsize
        assert xp.lib().xjh_paged_store(C.byref(kv.c), t, at, tok, at + 7 * buf.itemsize, tok, T, slot.ptr, None, err, 512) == 0
        xp.lib().xjh_sync()
        for off, got in zip((shift, shift + 7), kv.pages()):
            for i in range(T):
                want = buf[off + i * tok:off + i * tok + 128].astype(np.float16).reshape(2, 64)
                assert np.array_equal(got[i * 3 // 16, :, i * 3 % 16], want)


def test_store_refusals():
    L, err, one = xp.lib(), C.create_string_buffer(512), C.c_void_p(16)

    def store(type=xp.F16, Hkv=1, D=64, page=16, n_pages=2, k=16, v=16, bytes=1 << 20, rows=xp.F32, T=1, x=one, slot=one):
        c = xp.XjhPaged(type, Hkv, D, page, n_pages, k, v, bytes)
        return L.xjh_paged_store(C.byref(c), rows, x, 64, x, 64, T, slot, None, err, 512)

    for bad in ({"type": xp.F32}, {"type": xp.Q8_0}, {"Hkv": 0}, {"Hkv": 1025}, {"D": 96}, {"D": 512}, {"page": 8}, {"page": 24}, {"n_pages": 0}):
        assert store(**bad) == -1 and b"unsupported cache" in err.value, bad
    for bad in ({"k": None}, {"v": None}, {"k": 24}, {"v": 8}, {"bytes": 16 * 64 * 2 * 2 - 1}):
        assert store(**bad) == -1 and b"memory" in err.value, bad
    for bad in ({"rows": xp.BF16}, {"rows": xp.Q4_K}, {"T": -1}, {"T": (1 << 28) + 1}):
        assert store(**bad) == -1 and b"bad rows" in err.value, bad
    for bad in ({"x": None}, {"slot": None}):
        assert store(**bad) == -1 and b"no rows" in err.value, bad
    assert store(T=0, x=None, slot=None) == 0
    assert L.xjh_paged_store(None, xp.F32, one, 64, one, 64, 1, one, None, err, 512) == -1
    assert L.xjh_paged_bytes(None) == 0
