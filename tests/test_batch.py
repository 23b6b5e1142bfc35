"""The entries for several requests (xjh_page_plan, xjh_paged_store, xjh_attn_paged, xjh_attn_packed) against plain
forms written here from the text of xj_hip.h, and what they refuse (on the CPU, where nothing is launched).

Tables, lengths and slots are whole numbers and equal. A stored element is its row's, rounded once to nearest: equal bits.
Attention, with u the half step of the rows' type (f16 2^-11, bf16 2^-8): every weight is rounded once (u of it) and so is
the result, so an element is off by at most u of itself and u + 1e-5 of its row's sum_j p_j |v_j| (the 1e-5: fp32 sums and scores up to
20, off by a few of their own roundings: 20 * 1.44 * 4 * 2^-24 = 7e-6 in a weight). Float rows have no u, and 2e-6 over the norm of all rows, where
the roundings are independent.
"""
import ctypes as C

import numpy as np
import pytest

import xjpipe as xp
from test_long_context import Hip, rope64


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


@pytest.mark.gpu
@pytest.mark.parametrize("n_req,blocks", [(8, 8192), (8, 8193), (200, 500)])
def test_plan_small_steps_that_give_many_pages_back(n_req, blocks):
    """Long requests end while others take a token or a prompt, on both sides of 65536 pages."""
    L = blocks * 16
    pool, ref = xp.PagePool(16, n_req * blocks, n_req, blocks), RefPool(16, n_req * blocks, n_req, blocks)
    full = [L - 5 * r for r in range(n_req)]
    same_plan(pool, ref, n_past=[0] * n_req, n_new=full, T=50)
    end = [r % 4 != 1 for r in range(n_req)]
    past = [0 if e else n for e, n in zip(end, full)]
    got = same_plan(pool, ref, n_past=past, n_new=[17 if r == 2 else not e for r, e in enumerate(end)], held=full)
    assert got["status"][0] == 0 and pool.free.size > n_req * blocks // 2


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


def test_plan_refuses_lengths_where_it_writes():
    L, err = xp.lib(), C.create_string_buffer(512)
    at = {k: 4096 * (i + 1) for i, k in enumerate(("table", "free", "held", "past", "new", "n_free", "out", "cu", "kv", "pos", "slot", "status", "work"))}

    def plan(**to):
        b = {k: C.c_void_p(to.get(k, v)) for k, v in at.items()}
        p = xp.XjhPages(16, 8, 4, b["table"], b["free"])
        return L.xjh_page_plan(C.byref(p), b["held"], b["past"], b["new"], 5, b["n_free"], b["out"], 7, b["cu"], b["kv"], b["pos"], b["slot"], b["status"],
                               b["work"], 256, None, err, 512)

    sizes = {"out": 4, "cu": 24, "kv": 20, "pos": 28, "slot": 28, "status": 16, "work": 256, "table": 80, "free": 32}
    for n in ("held", "past", "new"):
        for k, size in sizes.items():
            for where in (at[k], at[k] + size - 4, at[k] - 16):
                assert plan(**{n: where}) == -1 and b"a buffer that is written" in err.value, (n, k)


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
    assert store(T=(1 << 26) + 1) == -1 and b"bad rows" in err.value
    for bad in ({"x": None}, {"slot": None}):
        assert store(**bad) == -1 and b"no rows" in err.value, bad
    assert store(T=0, x=None, slot=None) == 0
    assert L.xjh_paged_store(None, xp.F32, one, 64, one, 64, 1, one, None, err, 512) == -1
    assert L.xjh_paged_bytes(None) == 0


# -------------------------------------------------------------- attention --

IDS = {"f32": xp.F32, "f16": xp.F16, "bf16": xp.BF16}
HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def to_type(x, t):
    return bf16_bits(x) if t == "bf16" else x.astype(np.float16 if t == "f16" else np.float32)


def value(x):
    """The numbers that an array of float32, float16 or bf16 bits holds, in float64."""
    return (from_bf16(x) if x.dtype == np.uint16 else x).astype(np.float64)


def attend64(q, k, v, pos, seen=None, gate=None, window=0, n_sink=0, scale=None):
    """q [n][H][D] at positions pos .., k, v [m][Hkv][D], float64: (out, sum of p |v|). seen [m]: positions that exist."""
    n, H, D = q.shape
    m, G = k.shape[0], H // k.shape[1]
    p, j = pos + np.arange(n)[:, None], np.arange(m)[None]
    see = (j <= p) & ((window == 0) | (j > p - window) | (j < n_sink))
    if seen is not None:
        see = see & seen[None]
    out, mag = np.zeros((n, H, D)), np.zeros((n, H, D))
    for h in range(H):
        s = np.where(see, q[:, h] @ k[:, h // G].T * (D ** -0.5 if scale is None else scale), -np.inf)
        top = s.max(1, initial=-np.inf, keepdims=True)
        w = np.exp(s - np.where(np.isfinite(top), top, 0))
        w = np.divide(w, w.sum(1, keepdims=True), out=np.zeros_like(w), where=see.any(1, keepdims=True))
        out[:, h], mag[:, h] = w @ v[:, h // G], w @ np.abs(v[:, h // G])
        if gate is not None:
            sg = 1 / (1 + np.exp(-gate[:, h]))
            out[:, h], mag[:, h] = out[:, h] * sg, mag[:, h] * sg
    return out, mag


def check(got, want, mag, t):
    got = value(got).reshape(want.shape)
    u = HALF[t]
    assert np.all(np.isfinite(got))
    err, bar = np.abs(got - want), u * np.abs(want) + (u + 1e-5) * mag + (2.0 ** -24 if t == "f16" else 0)   # f16's smallest step
    assert np.all(err <= bar), (float((err / np.maximum(bar, 1e-300)).max()), np.unravel_index(np.argmax(err - bar), err.shape))
    if t == "f32" and np.linalg.norm(mag):
        assert np.linalg.norm(err) <= 2e-6 * np.linalg.norm(mag)


def kv_rows(rng, n, Hkv, D):
    x = rng.standard_normal((n, Hkv, D)) * np.exp(0.3 * rng.standard_normal((1, Hkv, D)) + 0.2 * rng.standard_normal((n, Hkv, 1)))
    return (x + 0.5 * rng.standard_normal((1, Hkv, D))).astype(np.float32)


class Batch:
    """Requests of (kv length, new rows) in shuffled pages whose other positions hold NaN."""

    def __init__(self, rng, lens, H, Hkv, D, page, rows="f16", cache="f16", spare=0, kv=None):
        self.lens, self.rows, self.D, self.H = lens, rows, D, H
        blocks = [up(max(n, 0), page) for n, _ in lens]
        n_pages = sum(blocks) + 2
        order = rng.permutation(n_pages)[:sum(blocks)].tolist()
        self.table = np.full((len(lens), max(blocks + [1]) + spare), -1, np.int32)
        nan = np.uint16(0x7E00 if cache == "f16" else 0x7FC0)
        pool = np.full((2, n_pages, Hkv, page, D), nan, np.uint16)
        self.kv = []
        for r, (n, _) in enumerate(lens):
            x = [to_type(a, cache) for a in (kv(r, n) if kv else (kv_rows(rng, n, Hkv, D), kv_rows(rng, n, Hkv, D)))]
            self.kv.append([value(a) for a in x])
            for b in range(blocks[r]):
                self.table[r, b] = g = order.pop()
                for w in range(2):
                    part = x[w][b * page:(b + 1) * page].view(np.uint16)
                    pool[w, g, :, :part.shape[0]] = part.transpose(1, 0, 2)
        self.cache = xp.PagedKv(Hkv, D, page, n_pages, type=IDS[cache])
        self.cache.k.put(pool[0]), self.cache.v.put(pool[1])
        self.cu = np.cumsum([0] + [m for _, m in lens])
        T = int(self.cu[-1])
        self.q, self.gate = (to_type((rng.standard_normal((T, H, D)) * 1.5).astype(np.float32), rows) for _ in range(2))

    def want(self, gate=False, **kw):
        got = []
        for r, (n, m) in enumerate(self.lens):
            rs = slice(int(self.cu[r]), int(self.cu[r + 1]))
            got.append(attend64(value(self.q[rs]), *self.kv[r], n - m, gate=value(self.gate[rs]) if gate else None, **kw))
        return tuple(np.concatenate([x[i] for x in got]) for i in range(2))

    def attend(self, gate=False, **kw):
        return self.cache.attend(self.q, self.table, self.cu, [n for n, _ in self.lens], gate=self.gate if gate else None, **kw)

    def check(self, max_new=None, work_bytes=None, **kw):
        got = self.attend(max_new=max_new, work_bytes=work_bytes, **kw)
        check(got, *self.want(**kw), self.rows)
        return got


EDGES = [(1, 1), (2, 1), (15, 1), (16, 2), (17, 3), (31, 1), (32, 4), (33, 1), (63, 2), (64, 1), (65, 5), (127, 1), (128, 1), (129, 1), (257, 7)]
PAIRS = [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [None, 0])   # few rows, many rows
@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 1, 128, 16), (16, 4, 256, 64), (8, 8, 64, 256), (15, 3, 64, 32), (6, 2, 128, 128), (3, 1, 256, 16)])
def test_paged_attention_of_few_rows(H, Hkv, D, page, rows, cache, max_new):
    b = Batch(np.random.default_rng(H + D), EDGES, H, Hkv, D, page, rows, cache)
    b.check(gate=True, max_new=1 if max_new is None else max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [None, 1])   # many rows, and the other kernel told wrongly
@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 1, 128, 16), (16, 4, 256, 64), (8, 8, 64, 256), (15, 3, 64, 32), (3, 1, 256, 16)])
def test_paged_attention_of_chunks(H, Hkv, D, page, rows, cache, max_new):
    lens = [(300, 300), (150, 33), (90, 90), (1, 1), (401, 129), (64, 64), (0, 0), (200, 0), (130, 1)]
    Batch(np.random.default_rng(H * D), lens, H, Hkv, D, page, rows, cache).check(max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (7, 4), (64, 0), (65, 64), (100, 130), (300, 2), (1 << 30, 5), ((1 << 31) - 1, 0), (50, (1 << 31) - 1)])
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 128), (4, 1, 64), (8, 2, 256)])
def test_paged_windows_and_first_tokens(H, Hkv, D, max_new, window, n_sink):
    """Positions behind the window are in no page."""
    lens = [(517, 1), (300, 6), (200, 70), (64, 64), (33, 1)]
    b = Batch(np.random.default_rng(window % 999), lens, H, Hkv, D, 16, "f32", "f16")
    for r, (n, m) in enumerate(lens):
        for i in range(up(n, 16)):
            if 16 * i + 15 <= n - m - window and 16 * i >= n_sink:
                b.table[r, i] = [-1, 1 << 30, -1 << 31][i % 3]
    b.check(window=window, n_sink=n_sink, max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("work_bytes", [None, 0, 64, 100000, 1 << 20])
def test_paged_splits(work_bytes, max_new, rows, cache):
    lens = [(5000, 1), (17, 1), (2100, 3), (640, 1), (1, 1)]
    Batch(np.random.default_rng(9), lens, 8, 2, 128, 32, rows, cache, spare=40).check(gate=True, max_new=max_new, work_bytes=work_bytes)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("n_req", [63, 64, 65, 300])
def test_paged_many_requests(n_req, max_new):
    rng = np.random.default_rng(n_req)
    lens = [(int(n), 1) for n in rng.integers(1, 700, n_req)]
    lens[n_req // 2] = (9000, 2)
    Batch(rng, lens, 4, 2, 64, 16, "bf16", "bf16").check(max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("work_bytes", [None, 0, 16, 200000])
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("rows,cache", [("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n_req,H,Hkv,D", [(250, 32, 8, 64), (40, 32, 32, 128), (70, 16, 4, 256)])
def test_paged_long_request_among_many_short_ones(n_req, H, Hkv, D, rows, cache, max_new, work_bytes):
    """More rows than the GPU holds at once, or than a wavefront looks at together; one of the requests is cut, in a mixed batch another of many rows too."""
    rng = np.random.default_rng(n_req)
    lens = [(int(n), 1) for n in rng.integers(1, 60, n_req)]
    lens[n_req // 3] = (6000, 1)
    if max_new == 0:
        lens[n_req // 2] = (1500, 40)
    Batch(rng, lens, H, Hkv, D, 32, rows, cache, spare=9).check(max_new=max_new, work_bytes=work_bytes)


def test_work_areas_serve_smaller_batches():
    """A work area asked for the largest step is as much as any smaller one's. A batch past the size at which the GPU is full without cutting has one too."""
    L, sizes = xp.lib(), [1, 2, 3, 8, 9, 30, 63, 64, 65, 103, 104, 105, 250, 505, 511, 512, 513, 1000, 1024, 1025, 3000, 9000]
    for t, H, Hkv, D in ((xp.BF16, 32, 8, 128), (xp.F32, 16, 4, 256), (xp.F16, 2, 1, 64), (xp.BF16, 16, 8, 128), (xp.F16, 32, 32, 64)):
        c = xp.XjhPaged(xp.F16 if t == xp.F32 else t, Hkv, D, 32, 1000, None, None, 0)
        paged = {}
        for most in (0, 1, 5, 100):
            n = paged[most] = [[L.xjh_attn_paged_work_bytes(C.byref(c), t, T, H, r, most, 4096) for T in sizes] for r in sizes]
            n = np.array(n, np.int64)
            assert n.min() > 0 and np.all(np.diff(n, axis=0) >= 0) and np.all(np.diff(n, axis=1) >= 0), (t, H, Hkv, D, most)
        n = np.array([[L.xjh_attn_packed_work_bytes(t, T, H, Hkv, D, r) for T in sizes] for r in sizes], np.int64)
        assert n[-1, -1] > 0 and np.all(np.diff(n, axis=0) >= 0) and np.all(np.diff(n, axis=1) >= 0), (t, H, Hkv, D)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
def test_paged_rows_before_the_first_position_and_of_no_request(max_new):
    """More new rows than positions: those before position 0 see nothing and are 0; rows past the last request keep their values."""
    rng, err = np.random.default_rng(3), C.create_string_buffer(512)
    b = Batch(rng, [(5, 5), (40, 3)], 4, 2, 64, 16, "f32", "f16")
    T, cu, kv = 12, np.array([0, 6, 9], np.int32), np.array([4, 40], np.int32)
    q = rng.standard_normal((T, 4, 64)).astype(np.float32)
    out = np.full((T, 4, 64), 7.0, np.float32)
    dq, do, dt, dc, dk = (xp.Dev(x) for x in (q, out, b.table, cu, kv))
    assert xp.lib().xjh_attn_paged(C.byref(b.cache.c), xp.F32, dq.ptr, 256, 64, None, 0, 0, dt.ptr, b.table.shape[1], dc.ptr, dk.ptr, 2, T, max_new, 4, 0, 0,
                                   0.125, do.ptr, 256, None, 0, None, err, 512) == 0
    xp.lib().xjh_sync()
    got = do.get(np.float32, out.shape)
    assert np.all(got[:2] == 0) and np.all(got[9:] == 7)
    w0 = attend64(q[2:6].astype(np.float64), b.kv[0][0][:4], b.kv[0][1][:4], 0)
    w1 = attend64(q[6:9].astype(np.float64), *b.kv[1], 37)
    check(got[2:6], *w0, "f32")
    check(got[6:9], *w1, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("cu,kv_len", [([0, 5, 3, 9], [20, 20, 20]), ([-4, 2, 100, 200], [20, 20, 20]), ([9, 0, 9, 9], [-3, 5, 1 << 30]),
                                       ([0, 3, 6, 9], [-1 << 31, 0, (1 << 31) - 1])])
def test_paged_lengths_that_make_no_sense_stay_in_bounds(cu, kv_len, max_new):
    b = Batch(np.random.default_rng(4), [(20, 3)] * 3, 2, 1, 64, 16)
    out = value(b.cache.attend(b.q, b.table, cu, kv_len, max_new=max_new))
    assert out.shape == (9, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_paged_values_that_are_not_finite(D, rows, cache, max_new):
    """Rows that do not see them are as without them; rows that do are not finite, in the dims concerned at least."""
    lens = [(90, 40), (70, 6), (33, 1)]
    for bad, at in ((np.inf, 60), (-np.inf, 75), (np.nan, 66)):
        def kv(r, n):
            rng = np.random.default_rng(r)
            return kv_rows(rng, n, 2, D), kv_rows(rng, n, 2, D)

        def spoilt(r, n):
            k, v = kv(r, n)
            if n > at:
                v[at, 1, D // 2 + 1] = bad
            return k, v

        clean = Batch(np.random.default_rng(1), lens, 4, 2, D, 16, rows, cache, kv=kv)
        b = Batch(np.random.default_rng(1), lens, 4, 2, D, 16, rows, cache, kv=spoilt)
        want, got = (value(x.attend(max_new=max_new)).reshape(-1, 4, D) for x in (clean, b))
        t = 0
        for n, m in lens:
            for p in range(n - m, n):
                hit = at < n and p >= at
                if hit:
                    assert not np.isfinite(got[t, 2:, D // 2 + 1]).any()
                    got[t, 2:, D // 2 + 1] = want[t, 2:, D // 2 + 1]
                assert np.array_equal(got[t], want[t]), (bad, n, p)
                t += 1


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("rows,cache", PAIRS)
def test_paged_keys_and_queries_that_are_not_finite(rows, cache, max_new):
    lens, D = [(80, 30), (50, 5)], 128
    def kv(r, n):
        rng = np.random.default_rng(r)
        return kv_rows(rng, n, 1, D), kv_rows(rng, n, 1, D)

    def spoilt(r, n):
        k, v = kv(r, n)
        k[47 + r, 0, 5] = np.nan
        return k, v

    clean = Batch(np.random.default_rng(1), lens, 2, 1, D, 32, rows, cache, kv=kv)
    b = Batch(np.random.default_rng(1), lens, 2, 1, D, 32, rows, cache, kv=spoilt)
    want, got = (value(x.attend(max_new=max_new)).reshape(-1, 2, D) for x in (clean, b))
    for t, (r, p) in enumerate([(r, p) for r, (n, m) in enumerate(lens) for p in range(n - m, n)]):
        if p >= 47 + r:
            assert not np.isfinite(got[t]).any()
        else:
            assert np.array_equal(got[t], want[t]), (r, p)
    q = clean.q.copy()
    q[7, 1, 3] = np.float32(np.inf) if rows == "f32" else {"f16": np.float16(np.inf), "bf16": np.uint16(0x7F80)}[rows]
    clean.q = q
    got = value(clean.attend(max_new=max_new)).reshape(-1, 2, D)
    assert not np.isfinite(got[7, 1]).any()
    got[7, 1] = want[7, 1]
    assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 4.0])
def test_paged_scales_of_any_sign(scale, max_new):
    """4.0: scores of some hundred, a weight each in 64 bits compared in norm by the rounding of such scores (2^-24 of 400 * 1.44, a few of them)."""
    b = Batch(np.random.default_rng(2), [(150, 40), (70, 1)], 4, 2, 64, 16, "f32", "f16")
    got, (want, mag) = b.attend(scale=scale, max_new=max_new), b.want(scale=scale)
    if scale != 4.0:
        check(got, want, mag, "f32")
    else:
        assert np.linalg.norm(value(got).reshape(want.shape) - want) <= 4 * 400 * 1.44 * 2.0 ** -24 * np.linalg.norm(mag)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e30])
def test_paged_float_queries_of_any_size(size, max_new):
    """Queries of a size and a scale that undoes it: the scores are ordinary."""
    for cache in ("f16", "bf16"):
        b = Batch(np.random.default_rng(2), [(150, 40), (70, 1)], 4, 2, 64, 16, "f32", cache)
        b.q = (b.q * np.float32(size)).astype(np.float32)
        b.check(scale=0.125 / size, max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
def test_paged_requests_that_share_pages(max_new):
    rng = np.random.default_rng(8)
    b = Batch(rng, [(100, 4), (100, 4), (40, 1)], 4, 1, 128, 16, "f16", "f16")
    b.table[1, :5], b.kv[1] = b.table[0, :5], [np.concatenate([x[:80], y[80:]]) for x, y in zip(b.kv[0], b.kv[1])]
    b.check(max_new=max_new)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new,work_bytes", [(1, None), (1, 0), (0, None)])
def test_paged_same_bits_again_and_in_any_batch(max_new, work_bytes):
    """The same call gives the same bits."""
    lens = [(3000, 1), (200, 60), (17, 3)]
    b = Batch(np.random.default_rng(2), lens, 8, 2, 128, 16, "bf16", "bf16")
    one = b.attend(max_new=max_new, work_bytes=work_bytes)
    for _ in range(3):
        assert np.array_equal(one, b.attend(max_new=max_new, work_bytes=work_bytes))


@pytest.mark.gpu
@pytest.mark.parametrize("others", [2, 80])
@pytest.mark.parametrize("rows,cache", PAIRS)
def test_paged_request_alone_and_in_any_batch(rows, cache, others):
    """A request's rows by themselves, in a batch, and with other kernels and work areas: each result is rounded once (u of it), weights are rounded to u in
    one kernel and not in the other (u of sum p |v|), and fp32 sums are 1e-5 of that apart from the exact ones, as above."""
    lens = [(3000, 1), (900, 60), (17, 3), (2500, 9)] + [(40, 1)] * others
    b = Batch(np.random.default_rng(2), lens, 8, 2, 128, 16, rows, cache)   # (60 tokens: 240 rows a kv head; 9: 36)
    want, mag = b.want()
    batches = [value(b.attend(max_new=m, work_bytes=w)).reshape(want.shape) for m, w in ((None, None), (0, None), (1, None), (None, 0), (1, 100000))]
    u, t = HALF[rows], 0
    for r, (n, m) in enumerate(lens[:5]):
        rs = slice(t, t + m)
        for most in (m, 0, 1):
            one = value(b.cache.attend(b.q[rs], b.table[r:r + 1], [0, m], [n], max_new=most)).reshape(m, 8, 128)
            for got in batches:
                assert np.all(np.abs(one - got[rs]) <= 2 * u * np.abs(want[rs]) + (u + 2e-5) * mag[rs] + (2.0 ** -24 if rows == "f16" else 0)), (r, most)
            if m * 4 <= 32 or most == 1:   # the kernel for few rows in both: no weights' rounding
                assert np.all(np.abs(one - batches[2][rs]) <= 2 * u * np.abs(want[rs]) + (u * u + 2e-5) * mag[rs] + (2.0 ** -24 if rows == "f16" else 0)), (r, most)
        t += m


PROMPTS = [300, 1, 0, 33, 128, 5, 129, 64, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D", [(2, 1, 128), (16, 4, 256), (8, 8, 64), (15, 3, 64), (3, 1, 256), (32, 8, 128)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (50, 3)])
def test_packed(H, Hkv, D, rows, window, n_sink):
    rng = np.random.default_rng(H + D)
    T, cu = sum(PROMPTS), np.cumsum([0] + PROMPTS)
    q, gate = (to_type((rng.standard_normal((T, H, D)) * 1.5).astype(np.float32), rows) for _ in range(2))
    k, v = (to_type(kv_rows(rng, T, Hkv, D), rows) for _ in range(2))
    got = xp.attn_packed(q, k, v, cu, gate=gate, window=window, n_sink=n_sink)
    w = [attend64(*(value(x[a:b]) for x in (q, k, v)), 0, gate=value(gate[a:b]), window=window, n_sink=n_sink) for a, b in zip(cu, cu[1:])]
    check(got, *(np.concatenate([x[i] for x in w]) for i in range(2)), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("work_bytes", [None, 0, 300000])
def test_packed_long(rows, work_bytes):
    rng = np.random.default_rng(1)
    T, H, Hkv, D = 2050, 2, 1, 64
    q = to_type((rng.standard_normal((T, H, D)) * 1.5).astype(np.float32), rows)
    k, v = (to_type(kv_rows(rng, T, Hkv, D), rows) for _ in range(2))
    got = xp.attn_packed(q, k, v, [0, 1900, T], work_bytes=work_bytes)
    w = [attend64(*(value(x[a:b]) for x in (q, k, v)), 0) for a, b in ((0, 1900), (1900, T))]
    check(got, *(np.concatenate([x[i] for x in w]) for i in range(2)), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D,shift,tok,head", [(64, 0, 0, 0), (64, 8, 16, 8), (128, 1, 3, 1), (128, 2, 8, 8), (256, 4, 8, 0), (64, 8, 1, 8)])
@pytest.mark.parametrize("lens", [(40, 1, 49), (1030, 3, 70)])
def test_packed_strides_and_alignment(lens, D, shift, tok, head, rows):
    """Rows that begin at any element, heads and tokens apart, q k v and gate in one buffer; what lies between is left alone."""
    rng, err = np.random.default_rng(5), C.create_string_buffer(512)
    H, Hkv, cu, T, n = 4, 2, np.cumsum((0,) + lens).astype(np.int32), sum(lens) + 3, sum(lens)
    hs = D + head
    ts = 2 * H * hs + 2 * Hkv * hs + tok
    buf = to_type(rng.standard_normal(shift + T * ts + 8 * D).astype(np.float32), rows)
    o_tok = H * D + 3
    out = np.full(T * o_tok, 9, buf.dtype)
    db, do, dc = xp.Dev(buf), xp.Dev(out), xp.Dev(cu)
    size = buf.itemsize
    at = [shift + x * hs for x in (0, H, H + Hkv, H + 2 * Hkv)]   # q, k, v, gate
    ptr = [db.ptr + x * size for x in at]
    wb = xp.lib().xjh_attn_packed_work_bytes(IDS[rows], T, H, Hkv, D, 3)
    work = xp.Dev(nbytes=max(16, wb))
    assert xp.lib().xjh_attn_packed(IDS[rows], ptr[0], ts, hs, ptr[1], ts, hs, ptr[2], ts, hs, ptr[3], ts, hs, dc.ptr, 3, T, H, Hkv, D, 0, 0,
                                    D ** -0.5, do.ptr, o_tok, work.ptr, wb, None, err, 512) == 0, err.value
    xp.lib().xjh_sync()
    got = do.get(buf.dtype, out.shape).reshape(T, o_tok)
    assert np.all(got[:, H * D:] == 9) and np.all(got[n:] == 9)
    def take(x, n):
        return value(np.stack([[buf[x + t * ts + h * hs:x + t * ts + h * hs + D] for h in range(n)] for t in range(T)]))

    q, k, v, g = take(at[0], H), take(at[1], Hkv), take(at[2], Hkv), take(at[3], H)
    w = [attend64(q[a:b], k[a:b], v[a:b], 0, gate=g[a:b]) for a, b in zip(cu, cu[1:])]
    check(np.ascontiguousarray(got[:n, :H * D]), *(np.concatenate([x[i] for x in w]) for i in range(2)), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T", [120, 1200])
def test_packed_values_that_are_not_finite(T, rows):
    """One prompt's do not reach another's rows, nor earlier ones of its own."""
    rng = np.random.default_rng(2)
    D, cu = 64, [0, 70, T]
    q = to_type(rng.standard_normal((T, 2, D)).astype(np.float32), rows)
    k, v = (kv_rows(rng, T, 1, D) for _ in range(2))
    want = value(xp.attn_packed(q, to_type(k, rows), to_type(v, rows), cu))
    v[50, 0, 9], k[110, 0, 3] = np.inf, np.nan
    got = value(xp.attn_packed(q, to_type(k, rows), to_type(v, rows), cu))
    assert not np.isfinite(got.reshape(T, 2, D)[50:70, :, 9]).any() and not np.isfinite(got[110:]).any()
    assert np.array_equal(got[:50], want[:50]) and np.array_equal(got[70:110], want[70:110])


def test_attention_refusals():
    L, err, one = xp.lib(), C.create_string_buffer(512), C.c_void_p(16)

    def paged(type=xp.F16, Hkv=2, D=64, page=16, n_pages=2, k=16, v=16, bytes=1 << 20, rows=xp.F32, q=one, out=one, table=one, blocks=4, cu=one,
              kv=one, n_req=1, T=1, H=4, window=0, n_sink=0, scale=1.0, work=None):
        c = xp.XjhPaged(type, Hkv, D, page, n_pages, k, v, bytes)
        return L.xjh_attn_paged(C.byref(c), rows, q, 256, 64, None, 0, 0, table, blocks, cu, kv, n_req, T, 1, H, window, n_sink, scale, out, 256,
                                work, 0, None, err, 512)

    for bad in ({"type": xp.F32}, {"Hkv": 0}, {"D": 32}, {"page": 1}, {"page": 512}, {"n_pages": 0}):
        assert paged(**bad) == -1 and b"unsupported cache" in err.value, bad
    for bad in ({"k": None}, {"v": 20}, {"bytes": 100}):
        assert paged(**bad) == -1 and b"memory" in err.value, bad
    for bad in ({"rows": xp.BF16}, {"rows": xp.Q8_0}, {"blocks": 0}, {"blocks": (1 << 26) + 1}, {"n_req": -1}, {"n_req": 65537}, {"T": -1}, {"T": 1 << 27},
                {"H": 3}, {"H": 0}, {"H": -2}, {"window": -1}, {"n_sink": -1}, {"scale": float("nan")}, {"scale": float("inf")}):
        assert paged(**bad) == -1 and b"bad shape" in err.value, bad
    for bad in ({"q": None}, {"out": None}, {"table": None}, {"cu": None}, {"kv": None}, {"work": C.c_void_p(8)}):
        assert paged(**bad) == -1 and b"buffer is missing" in err.value, bad
    assert paged(T=0, q=None) == 0 and paged(n_req=0, table=None) == 0
    for bad in ({"T": (1 << 25) + 1}, {"T": 65536, "n_req": 65536, "Hkv": 128, "H": 128, "bytes": 1 << 23}):   # more rows than a launch has room for
        assert paged(**bad) == -1 and b"bad shape" in err.value, bad

    def packed(type=xp.F32, q=one, k=one, v=one, out=one, cu=one, n=1, T=1, H=4, Hkv=2, D=64, window=0, n_sink=0, scale=1.0, work=None):
        return L.xjh_attn_packed(type, q, 256, 64, k, 128, 64, v, 128, 64, None, 0, 0, cu, n, T, H, Hkv, D, window, n_sink, scale, out, 256, work, 0, None,
                                 err, 512)

    for bad in ({"type": xp.Q8_0}, {"n": -1}, {"T": -1}, {"T": 1 << 27}, {"H": 3}, {"Hkv": 0}, {"Hkv": 1025, "H": 1025}, {"D": 80}, {"window": -1},
                {"n_sink": -2}, {"scale": float("-inf")}):
        assert packed(**bad) == -1 and b"bad shape" in err.value, bad
    for bad in ({"q": None}, {"k": None}, {"v": None}, {"out": None}, {"cu": None}, {"work": C.c_void_p(4)}):
        assert packed(**bad) == -1 and b"buffer is missing" in err.value, bad
    assert packed(T=0, q=None) == 0 and packed(n=0, cu=None) == 0
    c = xp.XjhPaged(xp.F16, 2, 64, 16, 2, None, None, 0)
    assert L.xjh_attn_paged_work_bytes(C.byref(c), xp.BF16, 1, 4, 1, 1, 4) == 0 and L.xjh_attn_packed_work_bytes(xp.F32, 1, 3, 2, 64, 1) == 0
    # enough for any smaller batch
    n = [L.xjh_attn_paged_work_bytes(C.byref(c), xp.F16, T, 4, T, 1, 4096) for T in (1, 2, 8, 64)]
    assert n[0] > 0 and n == sorted(n)


# --------------------------------------------------------------- together --

def _call(name, *args):
    err = C.create_string_buffer(512)
    assert getattr(xp.lib(), name)(*args, err, 512) == 0, err.value


class _Step:
    """A layer step of several requests on a stream, every length on the device: plan, rope of queries and keys at the plan's
    positions, store into the plan's slots, attention over the plan's table."""

    def __init__(self, n_req, T, H, Hkv, D, page, n_pages, blocks, rows="f32", cache="f16", max_new=0, window=0, n_sink=0):
        self.n_req, self.T, self.H, self.max_new, self.window, self.n_sink, self.blocks, self.rows = n_req, T, H, max_new, window, n_sink, blocks, rows
        self.pool = xp.PagePool(page, n_pages, n_req, blocks)
        self.kv = xp.PagedKv(Hkv, D, page, n_pages, type=IDS[cache])
        nan = np.full(self.kv.c.bytes // 2, 0x7FC0 if cache == "bf16" else 0x7E00, np.uint16)
        self.kv.k.put(nan), self.kv.v.put(nan)
        i32 = {"held": n_req, "past": n_req, "new": n_req, "cu": n_req + 1, "kv": n_req, "pos": T, "slot": T, "status": 4}
        self.d = {k: xp.Dev(np.zeros(n, np.int32)) for k, n in i32.items()}
        self.q, self.qr, self.k, self.kr, self.v, self.out = (xp.Dev(nbytes=4 * T * h * D) for h in (H, H, Hkv, Hkv, Hkv, H))
        self.cfg = xp.XjhRopeCfg(pairs=0, n_rot=D, base=1e4, scaling=0, factor=1.0)
        self.plan_bytes = xp.lib().xjh_page_plan_work_bytes(n_req)
        self.bytes = xp.lib().xjh_attn_paged_work_bytes(C.byref(self.kv.c), IDS[rows], T, H, n_req, max_new, blocks)
        self.plan_work, self.work = xp.Dev(nbytes=max(16, self.plan_bytes)), xp.Dev(nbytes=max(16, self.bytes))
        self.seen = [(np.zeros((0, Hkv, D)), np.zeros((0, Hkv, D))) for _ in range(n_req)]   # what every request's cache holds

    def run(self, st):
        d, c, T, H = {k: x.ptr for k, x in self.d.items()}, self.kv.c, self.T, self.H
        D, row, free = c.D, c.Hkv * c.D, self.pool._n_free.ptr
        _call("xjh_page_plan", C.byref(self.pool.p), d["held"], d["past"], d["new"], self.n_req, free, free, T, d["cu"], d["kv"], d["pos"], d["slot"],
              d["status"], self.plan_work.ptr, self.plan_bytes, st)
        for x, y, h in ((self.q, self.qr, H), (self.k, self.kr, c.Hkv)):
            _call("xjh_rope_scaled", x.ptr, h * D, D, y.ptr, h * D, D, T, h, D, C.byref(self.cfg), d["pos"], 0, st)
        _call("xjh_paged_store", C.byref(c), xp.F32, self.kr.ptr, row, self.v.ptr, row, T, d["slot"], st)
        _call("xjh_attn_paged", C.byref(c), xp.F32, self.qr.ptr, H * D, D, None, 0, 0, self.pool._table.ptr, self.blocks, d["cu"], d["kv"], self.n_req, T,
              self.max_new, H, self.window, self.n_sink, D ** -0.5, self.out.ptr, H * D, self.work.ptr, self.bytes, st)

    def feed(self, rng, held, past, new):
        for k, x in (("held", held), ("past", past), ("new", new)):
            self.d[k].put(np.asarray(x, np.int32))
        D, Hkv = self.kv.c.D, self.kv.c.Hkv
        self.x = [rng.standard_normal((self.T, h, D)).astype(np.float32) for h in (self.H, Hkv, Hkv)]
        for d, x in zip((self.q, self.k, self.v), self.x):
            d.put(x)
        self.out.put(np.full((self.T, self.H, D), 7, np.float32))

    def check(self, past, new):
        got, t = self.out.get(np.float32, (self.T, self.H, self.kv.c.D)), 0
        assert self.d["status"].get(np.int32, (4,)).tolist() == [0, 0, 0, sum(new)]
        for r, (p, n) in enumerate(zip(past, new)):
            pos = p + np.arange(n)
            q, k = (rope64(x[t:t + n], self.cfg, pos)[0].astype(np.float32) for x in self.x[:2])
            k, v = (np.concatenate([old[:p], value(to_type(x, "f16"))]) for old, x in zip(self.seen[r], (k, self.x[2][t:t + n])))
            self.seen[r] = k, v
            want, mag = attend64(q.astype(np.float64), k, v, p, window=self.window, n_sink=self.n_sink)
            # a key within half a bit of a border may round to the other side after the rotation: half a step of f16 in a few of a key's elements, each
            # 2^-11 of one of D products of a score of size 1, is below 2^-11 |q| / sqrt(D) in a score; as much of a weight
            err = np.abs(got[t:t + n] - want)
            assert np.all(err <= (1e-5 + 2.0 ** -11) * mag), (r, p, n, float((err / np.maximum(mag, 1e-30)).max()))
            assert np.linalg.norm(err) <= 2e-5 * max(np.linalg.norm(mag), 1e-30)
            t += n
        assert np.all(got[t:] == 7)   # the padding's rows


def _lengths(rng, n_req, T, limit, steps, most=None):
    """held, past, new of the steps of a batch: prompts, pieces of them, single tokens, rejected drafts, requests that end."""
    past, new = np.zeros(n_req, int), np.zeros(n_req, int)
    for _ in range(steps):
        held = past + new
        past = held - rng.integers(0, 3, n_req) * (rng.random(n_req) < 0.3)
        past[rng.random(n_req) < 0.1] = 0
        past = np.maximum(past, 0)
        new = np.where(rng.random(n_req) < 0.3, rng.integers(0, T // 2, n_req), rng.integers(0, 4, n_req))
        new = np.minimum(new, limit - past if most is None else most)
        while new.sum() > T:
            new[new.argmax()] //= 2
        yield held.tolist(), past.tolist(), new.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hkv,page,max_new,window,n_sink", [(128, 2, 16, 0, 0, 0), (64, 1, 32, 0, 40, 3), (256, 2, 64, 0, 0, 0), (128, 2, 16, 3, 0, 0)])
def test_captured_steps_of_a_batch(D, Hkv, page, max_new, window, n_sink):
    """Two steps captured once each, with work areas of their own, and replayed by turns over a batch's life, eager work between."""
    rng, hip = np.random.default_rng(D + page), Hip()
    steps = [_Step(5, 40, 2 * Hkv, Hkv, D, page, 5 * up(320, page), up(320, page), max_new=max_new, window=window, n_sink=n_sink) for _ in range(2)]
    streams = [hip.stream() for _ in steps]
    graphs = [hip.capture(st, s.run) for s, st in zip(steps, streams)]
    for i, (held, past, new) in enumerate(_lengths(rng, 5, 40, 320, 10, max_new or None)):
        for s in steps:
            s.feed(rng, held, past, new)
        hip.sync()
        for g, st in zip(graphs, streams):
            hip("hipGraphLaunch", g, st)
        xp.norm(rng.standard_normal((3, 64)).astype(np.float32), None, 1, 1e-6)
        hip.sync()
        for s in steps:
            s.check(past, new)
    for g in graphs:
        hip("hipGraphExecDestroy", g)
    for st in streams:
        hip("hipStreamDestroy", st)


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [60, 1, 0])   # 1: told wrongly
@pytest.mark.parametrize("slots", [70, 140])
def test_captured_step_of_many_slots(slots, max_new):
    """A step of 70 and of 140 slots, most of them idle: one request grows until it is cut, shrinks, ends and begins anew; replayed beside eager work. The attention is
    compared over the keys and values that lie in the pages: a key that the rotation's own rounding takes over a border of f16 moves the
    scores of a request of two or three positions by more than all else does. Those keys are their rotated rows', rounded once: half a step of f16, and
    the rotation's four roundings in fp32 of elements up to 6."""
    rng, hip = np.random.default_rng(70), Hip()
    s = _Step(slots, 90, 4, 2, 64, 16, slots * 40, 40, max_new=max_new)
    st = hip.stream()
    graph = hip.capture(st, s.run)
    past = np.zeros(slots, int)
    for i, grow in enumerate((60, 60, 60, 60, 1, 60, 60, 1, 1, 60, 1, 1, 0, 1, 50)):
        held = past.copy()
        if i == 8:
            past[17] -= 170
        if i == 12:
            past[17] = 0
        new = np.zeros(slots, int)
        new[rng.integers(0, slots, 25)] += 1
        new[17] = grow
        s.feed(rng, held.tolist(), past.tolist(), new.tolist())
        hip.sync()
        hip("hipGraphLaunch", graph, st)
        xp.norm(rng.standard_normal((3, 64)).astype(np.float32), None, 1, 1e-6)
        hip.sync()
        assert s.d["status"].get(np.int32, (4,)).tolist() == [0, 0, 0, new.sum()]
        got, q, table, pages = s.out.get(np.float32, (90, 4, 64)), s.qr.get(np.float32, (90, 4, 64)), s.pool.table, s.kv.pages()
        want, t = [], 0
        for r in np.flatnonzero(new):
            n, m = past[r] + new[r], new[r]
            k, v = (x[table[r, :up(n, 16)]].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:n].astype(np.float64) for x in pages)
            turned = rope64(s.x[1][t:t + m], s.cfg, past[r] + np.arange(m))[0]
            assert np.all(np.abs(k[past[r]:] - turned) <= 2.0 ** -11 * np.abs(turned) + 4 * 6 * 2.0 ** -24 + 2.0 ** -25)
            assert np.array_equal(v[past[r]:], s.x[2][t:t + m].astype(np.float16))
            assert np.all(np.abs(q[t:t + m] - rope64(s.x[0][t:t + m], s.cfg, past[r] + np.arange(m))[0]) <= 4 * 6 * 2.0 ** -24)
            want.append(attend64(q[t:t + m].astype(np.float64), k, v, past[r]))
            t += m
        check(got[:t], *(np.concatenate([x[i] for x in want]) for i in range(2)), "f32")
        assert np.all(got[t:] == 7)
        past = past + new
    hip("hipGraphExecDestroy", graph)
    hip("hipStreamDestroy", st)


@pytest.mark.gpu
@pytest.mark.parametrize("handle", [None, 1, 2])
def test_eager_steps_on_predefined_streams(handle):
    rng = np.random.default_rng(3)
    s = _Step(3, 24, 4, 2, 64, 16, 60, 20)
    for held, past, new in _lengths(rng, 3, 24, 320, 5):
        s.feed(rng, held, past, new)
        s.run(handle)
        xp.lib().xjh_sync()
        s.check(past, new)


@pytest.mark.gpu
def test_batch_calls_follow_their_stream():
    """Inputs that a side stream copies in behind half a gigabyte of other copies are there when the calls run."""
    rng, hip = np.random.default_rng(5), Hip()
    s = _Step(3, 24, 4, 2, 128, 16, 60, 20)
    s.feed(rng, [0, 0, 0], [0, 0, 0], [9, 1, 14])
    src, to = [xp.Dev(x) for x in s.x], (s.q, s.k, s.v)
    for d, x in zip(to, s.x):
        d.put(x * 0)
    big, st = [xp.Dev(nbytes=1 << 26) for _ in range(2)], hip.stream()
    hip.sync()
    for _ in range(8):
        hip("hipMemcpyAsync", C.c_void_p(big[0].ptr), C.c_void_p(big[1].ptr), C.c_size_t(1 << 26), C.c_int(3), st)
    for d, y in zip(to, src):
        hip("hipMemcpyAsync", C.c_void_p(d.ptr), C.c_void_p(y.ptr), C.c_size_t(y.nbytes), C.c_int(3), st)
    s.run(st)
    hip.sync()
    hip("hipStreamDestroy", st)
    s.check([0, 0, 0], [9, 1, 14])


@pytest.mark.gpu
@pytest.mark.parametrize("max_new", [1, 0])
def test_pages_beyond_four_gigabytes(max_new):
    """Requests in the last pages of caches of 5 GB each."""
    rng, Hkv, D, page, n_pages = np.random.default_rng(6), 8, 256, 256, 5000
    c = xp.XjhPaged(xp.BF16, Hkv, D, page, n_pages, 16, 16, 0)
    c.bytes = xp.lib().xjh_paged_bytes(C.byref(c))
    assert c.bytes > 1 << 32
    pool = [xp.Dev(nbytes=c.bytes) for _ in range(2)]
    c.k, c.v = pool[0].ptr, pool[1].ptr
    n, table = 700, np.array([[n_pages - 1, n_pages - 3, n_pages - 2]], np.int32)
    k, v = (to_type(kv_rows(rng, n, Hkv, D), "bf16") for _ in range(2))
    q = to_type(rng.standard_normal((40, Hkv, D)).astype(np.float32), "bf16")
    j = np.arange(n)
    slot = (table[0, j // page] * page + j % page).astype(np.int32)
    dk, dv, ds, dq, dt, dc, dl = (xp.Dev(x) for x in (k, v, slot, q, table, np.array([0, 40], np.int32), np.array([n], np.int32)))
    out, row = xp.Dev(nbytes=q.nbytes), Hkv * D
    nb = xp.lib().xjh_attn_paged_work_bytes(C.byref(c), xp.BF16, 40, Hkv, 1, max_new, 3)
    work = xp.Dev(nbytes=max(16, nb))
    _call("xjh_paged_store", C.byref(c), xp.BF16, dk.ptr, row, dv.ptr, row, n, ds.ptr, None)
    _call("xjh_attn_paged", C.byref(c), xp.BF16, dq.ptr, row, D, None, 0, 0, dt.ptr, 3, dc.ptr, dl.ptr, 1, 40, max_new, Hkv, 0, 0, D ** -0.5, out.ptr, row,
          work.ptr, nb, None)
    xp.lib().xjh_sync()
    check(out.get(np.uint16, q.shape), *attend64(value(q), value(k), value(v), n - 40), "bf16")
    for b in pool:
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_rows_of_more_than_two_billion_elements(packed):
    """A token of 2^23 heads of 256 and five more, all of one query: the same result in each, the last ones' too."""
    rng, hip, D, H, n = np.random.default_rng(7), Hip(), 256, (1 << 23) + 5, 20
    kv = xp.PagedKv(1, D, 32, 1)
    k, v = (kv_rows(rng, n, 1, D).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((1, 1, D)).astype(np.float16)
    if packed:
        k, v, n = k[:1], v[:1], 1
    kv.store(k, v, np.arange(n))
    dq, dk, dv, dt, dc, dl = (xp.Dev(x) for x in (q, k, v, np.zeros((1, 1), np.int32), np.array([0, 1], np.int32), np.array([n], np.int32)))
    out = xp.Dev(nbytes=2 * H * D)
    hip("hipMemset", C.c_void_p(out.ptr), C.c_int(0xFF), C.c_size_t(out.nbytes))
    if packed:
        _call("xjh_attn_packed", xp.F16, dq.ptr, D, 0, dk.ptr, D, D, dv.ptr, D, D, None, 0, 0, dc.ptr, 1, 1, H, 1, D, 0, 0, D ** -0.5, out.ptr, H * D,
              None, 0, None)
    else:
        _call("xjh_attn_paged", C.byref(kv.c), xp.F16, dq.ptr, D, 0, None, 0, 0, dt.ptr, 1, dc.ptr, dl.ptr, 1, 1, 1, H, 0, 0, D ** -0.5, out.ptr, H * D,
              None, 0, None)
    xp.lib().xjh_sync()
    got = out.get(np.float16, (H, D))
    check(got[:1], *attend64(value(q), value(k), value(v), n - 1), "f16")
    for i in range(0, H, 1 << 20):
        assert np.all(got[i:i + (1 << 20)].view(np.uint16) == got[0].view(np.uint16)), i


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D,at", [(64, 0), (128, 900), (256, 1199)])
def test_packed_long_prompt_among_empty_ones(D, at, rows):
    """A batch that may have more row tiles than the GPU holds and has a dozen: it is cut."""
    rng = np.random.default_rng(D)
    lens = np.zeros(1200, int)
    lens[[at, 500]] = 1500, 60
    T, cu = int(lens.sum()), np.cumsum(np.concatenate([[0], lens]))
    q = to_type((rng.standard_normal((T, 2, D)) * 1.5).astype(np.float32), rows)
    k, v = (to_type(kv_rows(rng, T, 1, D), rows) for _ in range(2))
    w = [attend64(*(value(x[a:b]) for x in (q, k, v)), 0) for a, b in zip(cu, cu[1:]) if b > a]
    for work_bytes in (None, 0, 500000):
        got = xp.attn_packed(q, k, v, cu, work_bytes=work_bytes)
        check(got, *(np.concatenate([x[i] for x in w]) for i in range(2)), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f16", "bf16", "f32"])
def test_packed_of_very_many_short_prompts(rows):
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 4, 3000)
    lens[[0, 1700]] = 70, 150
    T, cu = int(lens.sum()), np.cumsum(np.concatenate([[0], lens]))
    q, k, v = (to_type(rng.standard_normal((T, h, 64)).astype(np.float32), rows) for h in (4, 2, 2))
    got = xp.attn_packed(q, k, v, cu)
    w = [attend64(*(value(x[a:b]) for x in (q, k, v)), 0) for a, b in zip(cu, cu[1:])]
    check(got, *(np.concatenate([x[i] for x in w]) for i in range(2)), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("max_new", [1, 0])
def test_paged_rising_scores(rows, cache, max_new):
    """Scores that rise by some powers of two from tile to tile, and fall: the running maximum changes at every one, up to weights that vanish."""
    D, n = 64, 900
    for sign in (1, -1):
        def kv(r, m):
            rng = np.random.default_rng(4)
            k = np.zeros((m, 1, D))
            k[:, 0, 0] = sign * np.arange(m) / 4
            return (k + 0.1 * rng.standard_normal(k.shape)).astype(np.float32), rng.standard_normal((m, 1, D)).astype(np.float32)

        b = Batch(np.random.default_rng(4), [(n, 2), (n, 60)], 2, 1, D, 16, rows, cache, kv=kv)
        b.q = to_type(np.concatenate([np.ones((62, 2, 1)), 0.1 * np.random.default_rng(1).standard_normal((62, 2, D - 1))], -1).astype(np.float32), rows)
        # scores up to 225 of sums of that size: 225 * 1.44 * 4 * 2^-24 = 8e-5 in a weight beside what `check` allows
        got, (want, mag) = value(b.attend(scale=1.0, max_new=max_new)).reshape(-1, 2, D), b.want(scale=1.0)
        u = HALF[rows]
        assert np.all(np.abs(got - want) <= u * np.abs(want) + (u + 1e-4) * mag + 2.0 ** -24)


def _sized(rng, n, Hkv, D, size, scores):
    """Keys whose scores with queries of 1 in the first dim (0 elsewhere) are `scores` at scale 1, and values of that size, of one sign in the first half."""
    k = np.zeros((n, Hkv, D), np.float32)
    k[:, :, 0] = scores[:, None]
    v = (size * rng.uniform(0.5, 1, (n, Hkv, D))).astype(np.float32)
    v[:, :, D // 2:] *= np.where(rng.random((n, Hkv, D - D // 2)) < 0.5, -1, 1)
    return k, v


SCORES = {"equal": lambda n: np.zeros(n), "within the reference's tolerance": lambda n: np.where(np.arange(n) < 64, 0, 5.375)}


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("scores", SCORES)
@pytest.mark.parametrize("size", [2e38, 1e-30])
@pytest.mark.parametrize("max_new,work_bytes", [(1, None), (1, 0), (0, None), (0, 0)])
def test_paged_finite_values_of_any_size(max_new, work_bytes, size, scores, rows):
    """A mean of finite values is finite, and as near as that of ordinary ones. (1e-30 = 2^-100: what is lost below the smallest number, 2^-126, of
    900 products with weights of 2^-18 at least is 2^-26 of the result each, and they have the result's size together.)"""
    def kv(r, n):
        return _sized(np.random.default_rng(r), n, 2, 64, size, SCORES[scores](n))

    b = Batch(np.random.default_rng(1), [(900, 1), (900, 40), (3, 2)], 4, 2, 64, 16, rows, "bf16", kv=kv, spare=60)
    b.q = to_type(np.eye(1, 64, dtype=np.float32)[None].repeat(43, 0).repeat(4, 1), rows)
    b.check(scale=1.0, max_new=max_new, work_bytes=work_bytes)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,shift", [("f32", 0), ("bf16", 0), ("bf16", 1)])
@pytest.mark.parametrize("scores", SCORES)
@pytest.mark.parametrize("size", [2e38, 1e-30])
@pytest.mark.parametrize("lens,work", [((50, 14), True), ((900, 1100), True), ((900, 1100), False)])
def test_packed_finite_values_of_any_size(lens, work, size, scores, rows, shift):
    rng, T, H, Hkv, D = np.random.default_rng(2), sum(lens), 2, 1, 128
    q = to_type(np.eye(1, D, dtype=np.float32)[None].repeat(T, 0).repeat(H, 1), rows)
    kv = [_sized(rng, n, Hkv, D, size, SCORES[scores](n)) for n in lens]
    k, v = (to_type(np.concatenate([x[i] for x in kv]), rows) for i in range(2))
    pad = np.zeros(shift, q.dtype)
    dq, dk, dv, dc = (xp.Dev(x) for x in (q, np.concatenate([pad, k.ravel()]), np.concatenate([pad, v.ravel()]), np.cumsum((0,) + lens).astype(np.int32)))
    out, t = xp.Dev(nbytes=q.nbytes), IDS[rows]
    nb = xp.lib().xjh_attn_packed_work_bytes(t, T, H, Hkv, D, 2) if work else 0
    area, at = xp.Dev(nbytes=max(16, nb)), shift * q.itemsize
    _call("xjh_attn_packed", t, dq.ptr, H * D, D, dk.ptr + at, D, D, dv.ptr + at, D, D, None, 0, 0, dc.ptr, 2, T, H, Hkv, D, 0, 0, 1.0, out.ptr, H * D,
          area.ptr, nb, None)
    xp.lib().xjh_sync()
    w, lo = [], 0
    for n in lens:
        w.append(attend64(*(value(x[lo:lo + n]) for x in (q, k, v)), 0, scale=1.0))
        lo += n
    check(out.get(q.dtype, q.shape), *(np.concatenate([x[i] for x in w]) for i in range(2)), rows)


def test_batch_wrappers_refuse_arrays_of_other_shapes():
    x, kv = np.zeros((3, 2, 64), np.float32), xp.PagedKv.__new__(xp.PagedKv)   # (without memory: nothing is launched)
    kv.c = xp.XjhPaged(xp.F16, 2, 64, 16, 4, None, None, 0)
    tab = np.zeros((2, 3), np.int32)
    for call in (lambda: kv.store(x, x[:2], [0, 1, 2]), lambda: kv.store(x, x, [0, 1]), lambda: kv.store(x, x, [0, 1, 1]), lambda: kv.store(x, x.astype(np.float16), [0, 1, 2]),
                 lambda: kv.store(x.astype(np.float64), x, [0, 1, 2]), lambda: kv.store(x, x, [0, 1, 1 << 31]),
                 lambda: kv.attend(x[..., :32], tab, [0, 1, 3], [5, 5]), lambda: kv.attend(x, tab[0], [0, 1, 3], [5, 5]), lambda: kv.attend(x, tab, [0, 3], [5, 5]),
                 lambda: kv.attend(x, tab, [0, 1, 3], [5]), lambda: kv.attend(x, tab, [0, 1, 3], [5, 5], gate=x[:1]),
                 lambda: kv.attend(x, tab, [0, 1, 3], [5, 5], window=1 << 32), lambda: kv.attend(x, tab, [0, 1, 3], [5, 1 << 31]),
                 lambda: xp.attn_packed(x, x, x[:2], [0, 3]), lambda: xp.attn_packed(x, x.astype(np.float16), x, [0, 3]), lambda: xp.attn_packed(x, x, x, []),
                 lambda: xp.attn_packed(x, x, x, [0, 3], gate=x.astype(np.float16)), lambda: xp.attn_packed(x, x, x, [0, 3], n_sink=1 << 31),
                 lambda: xp.PagedKv(2, 60, 16, 4), lambda: xp.PagedKv(2, 64, 16, 4, type=xp.F32), lambda: xp.PagedKv(2, 64, 16, 1 << 31)):
        with pytest.raises(xp.XjError):
            call()
