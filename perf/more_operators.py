"""Cases of the operators for several requests at once: page tables, paged key/value cache, attention over ragged batches.

Kinds of case, and the calls behind them:

  plan    xjh_page_plan: pages taken and given back by request lengths, block tables, slots and positions of the new tokens
  store   xjh_paged_store: the keys and values of T new tokens into their slots
  paged   xjh_attn_paged: causal grouped-query attention of every request's new tokens over its pages, with or without
          a sliding window and first tokens that stay visible, with the sigmoid output gate
  packed  xjh_attn_packed: the same over whole prompts that lie one behind the other, keys and values as rows

Heads are those of the package's configurations (4B: 16 heads on 4 of 256, 0.8B: 8 on 2 of 256, tiny: 2 on 1 of 128)
and a few generic ones. Lengths come from the case alone; the seed orders them, and makes pages and values.
"""
import ctypes
import math
import os
import random
import sys
from types import SimpleNamespace

import torch

own = False
DEV = "cuda"
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
H4B, H08, TINY, GENERIC = {"H": 16, "Hkv": 4, "D": 256}, {"H": 8, "Hkv": 2, "D": 256}, {"H": 2, "Hkv": 1, "D": 128}, {"H": 32, "Hkv": 8, "D": 128}


def listed():
    return [
        # one decode step of a few requests: the smallest call, latency alone
        {"name": "plan_r8_decode", "kind": "plan", "page": 64, "n_req": 8, "past_lo": 1, "past_hi": 4000, "new_lo": 1, "new_hi": 1, "drop": 0.0, "mix": 1},
        # many requests, some ending or giving back rejected drafts, others with whole prompts
        {"name": "plan_r1000_ragged", "kind": "plan", "page": 16, "n_req": 1000, "past_lo": 1, "past_hi": 8000, "new_lo": 1, "new_hi": 700, "drop": 0.2, "mix": 2},
        # the rows of one decode step, two of them padding
        {"name": "store_f32_f16_4b_t16", "kind": "store", "rows": "f32", "cache": "f16", **H4B, "page": 64, "T": 16, "pad": 2},
        # the rows of long prompts
        {"name": "store_bf16_t8000", "kind": "store", "rows": "bf16", "cache": "bf16", **GENERIC, "page": 32, "T": 8000, "pad": 0},
        # one decoded token of one request of the small model: latency
        {"name": "paged_f16_tiny_r1_at_40", "kind": "paged", "rows": "f16", "cache": "f16", **TINY, "page": 16,
         "n_req": 1, "past_lo": 40, "past_hi": 40, "new_lo": 1, "new_hi": 1, "chunk_past": 0, "chunk_new": 0, "window": 0, "sinks": 0, "mix": 3},
        # one decoded token of a very long context: the cache's bytes
        {"name": "paged_f32_4b_r1_at_131000", "kind": "paged", "rows": "f32", "cache": "f16", **H4B, "page": 64,
         "n_req": 1, "past_lo": 131000, "past_hi": 131000, "new_lo": 1, "new_hi": 1, "chunk_past": 0, "chunk_new": 0, "window": 0, "sinks": 0, "mix": 4},
        # one decode step of many requests of very different lengths
        {"name": "paged_bf16_r64_decode", "kind": "paged", "rows": "bf16", "cache": "bf16", **GENERIC, "page": 32,
         "n_req": 64, "past_lo": 1, "past_hi": 16000, "new_lo": 1, "new_hi": 1, "chunk_past": 0, "chunk_new": 0, "window": 0, "sinks": 0, "mix": 5},
        # drafts of several requests verified, behind a window and four first tokens
        {"name": "paged_f32_4b_r8_t5_window", "kind": "paged", "rows": "f32", "cache": "f16", **H4B, "page": 128,
         "n_req": 8, "past_lo": 2000, "past_hi": 20000, "new_lo": 5, "new_hi": 5, "chunk_past": 0, "chunk_new": 0, "window": 2048, "sinks": 4, "mix": 6},
        # a step that takes a piece of one request's long prompt beside the others' single tokens
        {"name": "paged_bf16_4b_r32_chunk512_at_32000", "kind": "paged", "rows": "bf16", "cache": "bf16", **H4B, "page": 64,
         "n_req": 32, "past_lo": 100, "past_hi": 8000, "new_lo": 1, "new_hi": 1, "chunk_past": 32000, "chunk_new": 512, "window": 0, "sinks": 0, "mix": 7},
        # a few short prompts, one of them empty: latency
        {"name": "packed_f16_tiny_short", "kind": "packed", "rows": "f16", **TINY, "lens": "7+1+0+40+3", "window": 0, "sinks": 0},
        # ragged prompts as the layers here make them, in float
        {"name": "packed_f32_4b_2000", "kind": "packed", "rows": "f32", **H4B, "lens": "1100+333+500+3+64", "window": 0, "sinks": 0},
        # a long prompt with a short one behind it: the matrix cores' work
        {"name": "packed_bf16_8200", "kind": "packed", "rows": "bf16", **GENERIC, "lens": "8000+200", "window": 0, "sinks": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [H4B, H08, TINY, GENERIC, {"H": 8, "Hkv": 8, "D": 64}, {"H": 6, "Hkv": 2, "D": 128}, {"H": 15, "Hkv": 3, "D": 64}]


def draw(rng):
    kind = rng.choice(["plan", "store", "paged", "paged", "paged", "packed", "packed"])
    page, mix = rng.choice([16, 32, 64, 128, 256]), rng.randrange(1 << 30)
    if kind == "plan":
        n_req = _log_int(rng, 1, 1000)
        return {"kind": kind, "page": page, "n_req": n_req, "past_lo": 1, "past_hi": _log_int(rng, 2, 8000), "new_lo": 1,
                "new_hi": rng.choice([1, 5, _log_int(rng, 2, max(3, min(8000, 150000 // n_req)))]), "drop": rng.choice([0.0, 0.1, 0.3]), "mix": mix}
    rows, heads = rng.choice(["f32", "f16", "bf16"]), rng.choice(HEADS)
    windowed = rng.random() < 0.35
    c = {"kind": kind, "rows": rows, **heads}
    w = {"window": _log_int(rng, 1, 8192) if windowed else 0, "sinks": rng.choice([0, 1, 4, rng.randint(2, 150)]) if windowed else 0}
    if kind == "store":
        T = _log_int(rng, 1, 8000)
        return {**c, "cache": "f16" if rows == "f32" else rows, "page": page, "T": T, "pad": rng.choice([0, min(T, 3) - 1])}
    if kind == "paged":
        n_req = rng.choice([1, _log_int(rng, 2, 64)])
        new = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, max(10, 600 // n_req))])
        hi = max(4, min(131000, 1 << 19 if new < 9 else 1 << 15) // n_req)
        past = _log_int(rng, 2, hi)
        chunk = (_log_int(rng, 2, 32000) - 1, _log_int(rng, 9, 512)) if n_req > 1 and rng.random() < 0.3 else (0, 0)
        return {**c, "cache": "f16" if rows == "f32" else rows, "page": page, "n_req": n_req, "past_lo": rng.choice([1, past]), "past_hi": past,
                "new_lo": rng.choice([1, new]), "new_hi": new, "chunk_past": chunk[0], "chunk_new": chunk[1], **w, "mix": mix}
    left, lens = _log_int(rng, 1, 8000 if rows != "f32" else 2000), []
    while left > 0 and len(lens) < 40:
        n = min(left, _log_int(rng, 1, left))
        lens.append(n)
        left -= n
    return {**c, "lens": "+".join(map(str, lens + rng.choice([[], [0]]))), **w}


def _lengths(case):
    """[(n_past, n_new)] of the case's requests."""
    rng = random.Random(case["mix"])
    got = [(_log_int(rng, case["past_lo"], case["past_hi"]), _log_int(rng, case["new_lo"], case["new_hi"])) for _ in range(case["n_req"])]
    if case.get("chunk_new"):
        got[0] = case["chunk_past"], case["chunk_new"]
    return got


def _prompts(case):
    return [int(n) for n in case["lens"].split("+")]


def _plan_lengths(case):
    """[(held, n_past, n_new)]: requests that go on, that gave up drafts or that are over."""
    rng = random.Random(case["mix"] + 1)
    got = []
    for past, new in _lengths(case):
        x = rng.random() if case["drop"] else 1.0
        if x < case["drop"] / 2:
            got.append((past, 0, 0))
        elif x < case["drop"]:
            got.append((past + rng.randint(1, 40), past, new))
        else:
            got.append((0, 0, past) if case["new_hi"] > 8 and rng.random() < 0.1 else (past, past, new))
    return got


# ------------------------------------------------------------------- inputs --

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def _pages(n, page):
    return (n + page - 1) // page


def _like_rows(g, n, Hkv, D):
    """Keys or values [n][Hkv][D] as a layer makes them: channels of different size and mean, tokens of different size."""
    x = torch.randn(n, Hkv, D, generator=g, device=DEV)
    x *= torch.exp(0.3 * torch.randn(1, Hkv, D, generator=g, device=DEV)) * torch.exp(0.2 * torch.randn(n, Hkv, 1, generator=g, device=DEV))
    return x + 0.5 * torch.randn(1, Hkv, D, generator=g, device=DEV)


def _queries(g, case, T, i):
    qg = torch.randn(T, case["H"], 2 * case["D"], generator=g, device=DEV)   # [query | gate] of every head
    qg[..., :case["D"]] *= 1.5
    i.qg = qg.to(TYPE[case["rows"]])


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g, rng, i = _gen(seed), random.Random(seed), SimpleNamespace(case=case)
    if case["kind"] == "plan":
        P, lens = case["page"], _plan_lengths(case)
        rng.shuffle(lens)
        i.lens = lens
        have = [_pages(h, P) for h, _, _ in lens]
        need = [_pages(p + n, P) for _, p, n in lens]
        i.max_blocks = max(max(have), max(need))
        i.n_pages = sum(have) + sum(max(0, b - a) for a, b in zip(have, need)) + 100
        order = list(range(i.n_pages))
        rng.shuffle(order)
        table = [[-1] * i.max_blocks for _ in lens]
        for row, n in zip(table, have):
            row[:n] = [order.pop() for _ in range(n)]
        i.table, i.free, i.n_free = _ints(table), _ints(order + [-1] * (i.n_pages - len(order))), _ints([len(order)])
        i.held, i.n_past, i.n_new = (_ints([x[k] for x in lens]) for k in range(3))
        i.T = (sum(n for _, _, n in lens) + 7) // 8 * 8   # the step's rows, padded as a captured graph's
        return i
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["kind"] == "packed":
        lens = _prompts(case)
        rng.shuffle(lens)
        i.lens, T = lens, sum(lens)
        i.k, i.v = (_like_rows(g, T, Hkv, D).to(TYPE[case["rows"]]) for _ in range(2))
        _queries(g, case, T, i)
        i.cu = _ints([sum(lens[:n]) for n in range(len(lens) + 1)])
        return i
    P = case["page"]
    if case["kind"] == "store":
        T = case["T"]
        i.n_pages = _pages(T, P) + 5
        start = [p * P + o for p in torch.randperm(i.n_pages, generator=g, device=DEV).tolist()[:_pages(T, P)] for o in range(P)][:T]
        for t in rng.sample(range(T), case["pad"]):
            start[t] = -1
        i.slot = _ints(start)
        i.k_new, i.v_new = (_like_rows(g, T, Hkv, D).reshape(T, Hkv * D).to(TYPE[case["rows"]]) for _ in range(2))
        # one page more than the library is told of: the plain form's place for rows without a slot
        i.k, i.v = (torch.randn(i.n_pages + 1, Hkv, P, D, generator=g, device=DEV).to(TYPE[case["cache"]]) for _ in range(2))
        return i
    i.lens = _lengths(case)
    rng.shuffle(i.lens)
    blocks = [_pages(p + n, P) for p, n in i.lens]
    i.n_pages, i.max_blocks = sum(blocks) + 3, max(blocks)
    order = torch.randperm(i.n_pages, generator=g, device=DEV).tolist()
    i.table = _ints([[order.pop() for _ in range(b)] + [-1] * (i.max_blocks - b) for b in blocks])
    i.k, i.v = (_like_rows(g, i.n_pages * P, Hkv, D).reshape(i.n_pages, P, Hkv, D).transpose(1, 2).contiguous().to(TYPE[case["cache"]])
                for _ in range(2))
    i.cu = _ints([sum(n for _, n in i.lens[:r]) for r in range(len(i.lens) + 1)])
    i.kv_len = _ints([p + n for p, n in i.lens])
    _queries(g, case, sum(n for _, n in i.lens), i)
    return i


def prepare(case, seed):
    i = _inputs(case, seed)
    if case["kind"] == "plan":
        n, T = case["n_req"], i.T
        i.cu, i.kv_len, i.pos, i.slot, i.n_free_out, i.status = (torch.empty(m, dtype=torch.int32, device=DEV) for m in (n + 1, n, T, T, 1, 4))
    elif case["kind"] != "store":
        i.out = torch.empty(i.qg.shape[0], case["H"] * case["D"], dtype=i.qg.dtype, device=DEV)
    return i


# -------------------------------------------------------------- plain forms --

def _plan_answer(i):
    return {"table": i.table, "free": i.free, "n_free": i.n_free_out, "cu": i.cu, "kv_len": i.kv_len, "pos": i.pos, "slot": i.slot,
            "status": i.status}


def _plain_plan(i):
    P, T, L = i.case["page"], i.T, i.max_blocks * i.case["page"]
    past, new, held = i.n_past.long().clamp(0, L), i.n_new.long().clamp(min=0), i.held.long().clamp(0, L)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    cu = torch.cat([zero, new.cumsum(0)])
    kv = (past + new).clamp(max=L)
    have, need = (held + P - 1) // P, (kv + P - 1) // P
    rel, take = (have - need).clamp(min=0), (need - have).clamp(min=0)
    rel_cu, take_cu = torch.cat([zero, rel.cumsum(0)]), torch.cat([zero, take.cumsum(0)])
    n_free = i.n_free.long().clamp(0, i.n_pages)
    total = (n_free + rel_cu[-1]).clamp(max=i.n_pages)   # [1]
    k = torch.arange(i.n_pages, device=DEV)
    r = torch.searchsorted(rel_cu[1:], k - n_free, right=True).clamp(max=len(past) - 1)
    given = i.table[r, (need[r] + k - n_free - rel_cu[r]).clamp(0, i.max_blocks - 1)]
    stack = torch.where(k < n_free, i.free, given)                          # the free pages, then the released ones
    enough = take_cu[-1] <= total                                           # else none is taken
    left = torch.where(enough, total - take_cu[-1], total)
    b = torch.arange(i.max_blocks, device=DEV)[None]
    src = total - 1 - (take_cu[:-1, None] + b - have[:, None])
    page = torch.where(enough, stack[src.clamp(0, i.n_pages - 1)], -1)
    taking = (b >= have[:, None]) & (b < need[:, None])
    i.table.copy_(torch.where(taking, page, i.table))
    i.free.copy_(torch.where((k >= n_free) & (k < left), stack, i.free))
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True)
    real = r < len(past)
    r = r.clamp(max=len(past) - 1)
    pos = past[r] + t - cu[r]
    page = i.table[r, (pos // P).clamp(0, i.max_blocks - 1)].long()
    i.pos.copy_(torch.where(real, pos, 0))
    i.slot.copy_(torch.where(real & (pos < L) & (page >= 0) & (page < i.n_pages), page * P + pos % P, -1))
    i.cu.copy_(cu)
    i.kv_len.copy_(kv)
    i.n_free_out.copy_(left)
    i.status.copy_(torch.stack([(take_cu[-1] - total[0]).clamp(min=0), (past + new - L).clamp(min=0).sum(), (cu[-1] - T).clamp(min=0), cu[-1]]))
    return _plan_answer(i)


def _plain_store(i):
    P, T = i.case["page"], i.case["T"]
    slot = i.slot.long()
    page, at = torch.where(slot >= 0, slot // P, i.n_pages), torch.where(slot >= 0, slot % P, 0)
    for pool, new in ((i.k, i.k_new), (i.v, i.v_new)):
        pool[page, :, at] = new.float().reshape(T, i.case["Hkv"], i.case["D"]).to(pool.dtype)
    return {"k": i.k[:i.n_pages], "v": i.v[:i.n_pages]}


def _attend(case, q, gate, k, v, n_past):
    """q, gate [n][H][D] over k, v [m][Hkv][D], row t at position n_past + t; all float32."""
    n, H, D = q.shape
    Hkv, G, W = case["Hkv"], H // case["Hkv"], case["window"]
    p = n_past + torch.arange(n, device=DEV)[:, None]
    j = torch.arange(k.shape[0], device=DEV)
    see = j <= p
    if W:
        see &= (j > p - W) | (j < case["sinks"])
    out = torch.empty(n, H, D, device=DEV)
    q, k, v = (q * D ** -0.5).reshape(n, Hkv, G, D).permute(1, 2, 0, 3), k.permute(1, 2, 0), v.transpose(0, 1)
    step = max(1, (1 << 28) // (G * n * k.shape[2]))   # kv heads whose scores are 1 GB
    for h in range(0, Hkv, step):
        s = torch.matmul(q[h:h + step].reshape(-1, G * n, D), k[h:h + step].contiguous()).reshape(-1, G, n, k.shape[2])
        s.masked_fill_(~see, -math.inf)
        s = s.sub_(s.amax(-1, keepdim=True)).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.reshape(-1, G * n, k.shape[2]), v[h:h + step].contiguous()).reshape(-1, G, n, D) / total
        out[:, h * G:(h + step) * G] = o.permute(2, 0, 1, 3).reshape(n, -1, D)
    return out / (1 + torch.exp(-gate))


def _plain_attention(i):
    case, D = i.case, i.case["D"]
    out, t = torch.empty(i.qg.shape[0], case["H"], D, device=DEV), 0
    for r, ln in enumerate(i.lens):
        past, n = ln if case["kind"] == "paged" else (0, ln)
        if not n:
            continue
        if case["kind"] == "paged":
            row = i.table[r, :_pages(past + n, case["page"])].long()
            k, v = (x[row].transpose(1, 2).reshape(-1, case["Hkv"], D)[:past + n].float() for x in (i.k, i.v))
        else:
            k, v = i.k[t:t + n].float(), i.v[t:t + n].float()
        out[t:t + n] = _attend(case, i.qg[t:t + n, :, :D].float(), i.qg[t:t + n, :, D:].float(), k, v, past)
        t += n
    return out.reshape(t, -1).to(i.qg.dtype)


# ------------------------------------------------------- the library's calls --

def _lib():
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "meta-work_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import xjpipe
    return xjpipe


_err = ctypes.create_string_buffer(512)


def _work_area(i, n):
    i.work = torch.empty(max(1, n), dtype=torch.uint8, device=DEV)
    return i.work.data_ptr() if n else None, n


def _call(i):
    """The pass's library call, its arguments up to the stream, as a program keeps them, and what it returns."""
    xp, case = _lib(), i.case
    L, kind = xp.lib(), case["kind"]
    ids = {"f32": xp.F32, "f16": xp.F16, "bf16": xp.BF16}
    if kind == "plan":
        p = ctypes.pointer(xp.XjhPages(page=case["page"], n_pages=i.n_pages, max_blocks=i.max_blocks, table=i.table.data_ptr(),
                                       free_list=i.free.data_ptr()))
        at = [x.data_ptr() for x in (i.cu, i.kv_len, i.pos, i.slot, i.status)]
        return _plan_answer(i), L.xjh_page_plan, (p, i.held.data_ptr(), i.n_past.data_ptr(), i.n_new.data_ptr(), case["n_req"],
                                                  i.n_free.data_ptr(), i.n_free_out.data_ptr(), i.T, *at,
                                                  *_work_area(i, L.xjh_page_plan_work_bytes(case["n_req"])))
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if kind != "packed":
        c = ctypes.pointer(xp.XjhPaged(type=ids[case["cache"]], Hkv=Hkv, D=D, page=case["page"], n_pages=i.n_pages, k=i.k.data_ptr(),
                                       v=i.v.data_ptr(), bytes=i.k[:i.n_pages].numel() * 2))
    if kind == "store":
        return {"k": i.k[:i.n_pages], "v": i.v[:i.n_pages]}, L.xjh_paged_store, (
            c, ids[case["rows"]], i.k_new.data_ptr(), Hkv * D, i.v_new.data_ptr(), Hkv * D, case["T"], i.slot.data_ptr())
    T, q = i.qg.shape[0], i.qg.data_ptr()
    gate = q + D * i.qg.element_size()
    rows = (q, 2 * H * D, 2 * D), (gate, 2 * H * D, 2 * D)
    if kind == "paged":
        new = max(n for _, n in i.lens)
        work = _work_area(i, L.xjh_attn_paged_work_bytes(c, ids[case["rows"]], T, H, len(i.lens), new, i.max_blocks))
        return i.out, L.xjh_attn_paged, (c, ids[case["rows"]], *rows[0], *rows[1], i.table.data_ptr(), i.max_blocks, i.cu.data_ptr(),
                                         i.kv_len.data_ptr(), len(i.lens), T, new, H, case["window"], case["sinks"], D ** -0.5,
                                         i.out.data_ptr(), H * D, *work)
    work = _work_area(i, L.xjh_attn_packed_work_bytes(ids[case["rows"]], T, H, Hkv, D, len(i.lens)))
    return i.out, L.xjh_attn_packed, (ids[case["rows"]], *rows[0], i.k.data_ptr(), Hkv * D, D, i.v.data_ptr(), Hkv * D, D, *rows[1],
                                      i.cu.data_ptr(), len(i.lens), T, H, Hkv, D, case["window"], case["sinks"], D ** -0.5,
                                      i.out.data_ptr(), H * D, *work)


def _own(i):
    if not hasattr(i, "call"):
        i.answer, i.call, i.args = _call(i)
    if i.call(*i.args, torch.cuda.current_stream().cuda_stream, _err, 512) != 0:
        raise RuntimeError(_err.value.decode(errors="replace"))
    return i.answer


def run(i):
    if own:
        return _own(i)
    return {"plan": _plain_plan, "store": _plain_store, "paged": _plain_attention, "packed": _plain_attention}[i.case["kind"]](i)


# ------------------------------------------------------------------- bounds --

def _pairs(case, past, n):
    """(query, key) pairs of n rows behind `past` positions, and the positions that any of them sees."""
    W, S = case["window"], case["sinks"]
    if not n:
        return 0, 0
    if not W:
        return n * past + n * (n + 1) // 2, past + n
    first = (torch.arange(past, past + n, dtype=torch.int64) - W + 1).clamp(min=0)
    p = torch.arange(past, past + n, dtype=torch.int64)
    return int((p + 1 - first + first.clamp(max=S)).sum()), past + n - int(first[0]) + min(S, int(first[0]))


def work(case):
    if case["kind"] == "plan":
        P, lens = case["page"], _plan_lengths(case)
        moved = sum(abs(_pages(p + n, P) - _pages(h, P)) for h, p, n in lens)
        tokens = sum(n for _, _, n in lens)
        return {"bytes": 20 * len(lens) + 8 * moved + 8 * tokens, "flops": 4 * tokens + 8 * len(lens)}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    size = 4 if case["rows"] == "f32" else 2
    if case["kind"] == "store":
        n = (case["T"] - case["pad"]) * Hkv * D * 2
        return {"bytes": n * (size + 2) + 4 * case["T"], "flops": n}
    lens = _lengths(case) if case["kind"] == "paged" else [(0, n) for n in _prompts(case)]
    both = [_pairs(case, p, n) for p, n in lens]
    T = sum(n for _, n in lens)
    kv = 2 * Hkv * D * (2 if case["kind"] == "paged" else size)
    return {"bytes": kv * sum(s for _, s in both) + 3 * size * T * H * D, "flops": 4 * H * D * sum(p for p, _ in both)}


# ----------------------------------------------------------- 64-bit results --

def _exact_plan(case, i):
    """Request by request, page by page."""
    P, L = case["page"], i.max_blocks * case["page"]
    table, free = i.table.tolist(), i.free.tolist()
    stack = free[:i.n_free.item()]
    cu, kv_len, pos, slot = [0], [], [], []
    for (held, past, new), row in zip(i.lens, table):
        kv_len.append(min(past + new, L))
        stack += row[_pages(kv_len[-1], P):_pages(held, P)]
    missing = max(0, sum(max(0, _pages(n, P) - _pages(held, P)) for (held, _, _), n in zip(i.lens, kv_len)) - len(stack))
    for (held, past, new), row, n in zip(i.lens, table, kv_len):
        for b in range(_pages(held, P), _pages(n, P)):
            row[b] = -1 if missing else stack.pop()
        cu.append(cu[-1] + new)
        pos += range(past, past + new)
        slot += [row[p // P] * P + p % P if p < L and row[p // P] >= 0 else -1 for p in range(past, past + new)]
    n = i.n_free.item()
    free[n:len(stack)] = stack[n:]
    pad = i.T - len(pos)
    d = {"table": table, "free": free, "n_free": [len(stack)], "cu": cu, "kv_len": kv_len, "pos": pos + [0] * pad, "slot": slot + [-1] * pad,
         "status": [missing, sum(max(0, p + n - L) for _, p, n in i.lens), 0, cu[-1]]}
    return {k: _ints(v) for k, v in d.items()}


def _exact_store(case, i):
    out = {}
    for name, pool, new in (("k", i.k, i.k_new), ("v", i.v, i.v_new)):
        x = pool[:i.n_pages].double().transpose(1, 2).reshape(-1, case["Hkv"], case["D"])
        rows = torch.nonzero(i.slot >= 0)[:, 0]
        x[i.slot[rows].long()] = new[rows].double().reshape(-1, case["Hkv"], case["D"])
        out[name] = x.reshape(i.n_pages, case["page"], case["Hkv"], case["D"]).transpose(1, 2)
    return out


def _exact_attention(case, i):
    D, G, W, t0 = case["D"], case["H"] // case["Hkv"], case["window"], 0
    out = torch.empty(i.qg.shape[0], case["H"], D, dtype=torch.float64, device=DEV)
    for r, ln in enumerate(i.lens):
        past, n = ln if case["kind"] == "paged" else (0, ln)
        j = torch.arange(past + n, device=DEV)
        for h in range(case["H"]):
            if case["kind"] == "paged":
                page, at = i.table[r, j // case["page"]].long(), j % case["page"]
                k, v = i.k[page, h // G, at].double(), i.v[page, h // G, at].double()
            else:
                k, v = i.k[t0:t0 + n, h // G].double(), i.v[t0:t0 + n, h // G].double()
            for t in range(0, n, 512):
                rows = slice(t0 + t, t0 + min(t + 512, n))
                p = past + torch.arange(t, min(t + 512, n), device=DEV)[:, None]
                m = (j <= p) & ((j >= p - W + 1) | (j < case["sinks"]) | (W == 0))
                s = (i.qg[rows, h, :D].double() @ k.t().contiguous()) / math.sqrt(D)
                out[rows, h] = torch.softmax(torch.where(m, s, -math.inf), -1) @ v * torch.sigmoid(i.qg[rows, h, D:].double())
        t0 += n
    return out.reshape(t0, -1)


def exact(case, seed):
    i = _inputs(case, seed)
    return {"plan": _exact_plan, "store": _exact_store, "paged": _exact_attention, "packed": _exact_attention}[case["kind"]](case, i)
