"""Cases of the long-context operators: scaled rotary positions, the 8-bit key/value cache and attention over it.

Kinds of case, and the calls behind them:

  rope    xjh_rope_scaled: queries or keys of T tokens rotated into another buffer (half or interleaved
          pairs, part of the head, plain, linear or YaRN frequencies)
  store   xjh_kv8_store of T new rows behind n_past older ones, then xjh_kv8_load of every block that the
          rows touch (so the answer is the values that the codes stand for)
  load    xjh_kv8_load of a range of positions
  attn    xjh_attn_kv8: causal grouped-query attention of T tokens over the cache, with or without a
          sliding window and first tokens that stay visible, with the sigmoid output gate

Heads and sizes are those of the package's configurations (4B: 16 heads on 4 of 256, 0.8B: 8 on 2 of 256,
tiny: 2 on 1 of 128) and a few generic ones. The cache's codes are made here with plain torch, in position
order (`codes`, what the plain forms read) and in the cache's documented order (`cache`, what a program that
uses the library holds).
"""
import ctypes
import math
import os
import sys
from types import SimpleNamespace

import torch

own = False
DEV = "cuda"
I8, E4M3 = 0, 1
TYPE = {"i8": I8, "e4m3": E4M3}
LINEAR, YARN = 1, 2
SCALING = {"plain": 0, "linear": LINEAR, "yarn": YARN}


def listed():
    h4b, h08, tiny = {"H": 16, "Hkv": 4, "D": 256}, {"H": 8, "Hkv": 2, "D": 256}, {"H": 2, "Hkv": 1, "D": 128}
    return [
        # the queries of one decoded token far into an extended context: the smallest call, latency alone
        {"name": "rope_4b_q_t1_yarn", "kind": "rope", "heads": 16, "D": 256, "n_rot": 64, "pairs": "half", "scaling": "yarn",
         "pos0": 100001, "T": 1},
        # the queries of a long prompt, every dim rotated, interleaved pairs
        {"name": "rope_t4096_interleaved", "kind": "rope", "heads": 16, "D": 256, "n_rot": 256, "pairs": "interleaved",
         "scaling": "linear", "pos0": 28000, "T": 4096},
        # one decoded token written into a block that earlier tokens began
        {"name": "store_i8_4b_t1_at_4003", "kind": "store", "type": "i8", **h4b, "block": 32, "n_past": 4003, "T": 1},
        # a prompt piece written behind a ragged prefix
        {"name": "store_e4m3_4b_t2048_at_1001", "kind": "store", "type": "e4m3", **h4b, "block": 64, "n_past": 1001, "T": 2048},
        # a few positions of a small cache read back
        {"name": "load_e4m3_tiny_77", "kind": "load", "type": "e4m3", **tiny, "block": 16, "pos0": 5, "n": 77},
        # a long cache read back whole
        {"name": "load_i8_4b_32000", "kind": "load", "type": "i8", **h4b, "block": 64, "pos0": 0, "n": 32000},
        # one decoded token of the small model, short context: latency
        {"name": "attn_i8_tiny_t1_at_40", "kind": "attn", "type": "i8", **tiny, "block": 32, "n_past": 40, "T": 1, "window": 0, "sinks": 0},
        # one decoded token deep into the default 4096-token context
        {"name": "attn_i8_4b_t1_at_4000", "kind": "attn", "type": "i8", **h4b, "block": 32, "n_past": 4000, "T": 1, "window": 0, "sinks": 0},
        # one decoded token of a very long context: the cache's bytes
        {"name": "attn_e4m3_4b_t1_at_131000", "kind": "attn", "type": "e4m3", **h4b, "block": 64, "n_past": 131000, "T": 1, "window": 0, "sinks": 0},
        # a five-row verification behind a long prefix seen through a window and four first tokens
        {"name": "attn_i8_4b_t5_at_32003_window", "kind": "attn", "type": "i8", **h4b, "block": 32, "n_past": 32003, "T": 5, "window": 4096, "sinks": 4},
        # a ragged prompt chunk of the 0.8B shape with a window, one scale per token
        {"name": "attn_e4m3_0_8b_t333_at_7001", "kind": "attn", "type": "e4m3", **h08, "block": 1, "n_past": 7001, "T": 333, "window": 1024, "sinks": 4},
        # a whole prompt of the 4B shape: the matrix cores' work
        {"name": "attn_i8_4b_t2048_at_0", "kind": "attn", "type": "i8", **h4b, "block": 64, "n_past": 0, "T": 2048, "window": 0, "sinks": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(16, 4, 256), (8, 2, 256), (2, 1, 128), (8, 8, 64), (6, 2, 128), (16, 2, 64)]


def draw(rng):
    kind = rng.choice(["rope", "store", "load", "attn", "attn", "attn"])
    if kind == "rope":
        D = rng.choice([64, 128, 256])
        heads = rng.choice([1, 2, 4, 8, 16])
        return {"kind": kind, "heads": heads, "D": D, "n_rot": rng.choice([D, D // 2, D // 4, 2 * rng.randint(1, D // 2)]),
                "pairs": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["plain", "linear", "yarn"]),
                "pos0": _log_int(rng, 1, 1 << 20), "T": _log_int(rng, 1, 4096 * 16 * 256 // (heads * D) // 4)}
    H, Hkv, D = rng.choice(HEADS)
    c = {"kind": kind, "type": rng.choice(["i8", "e4m3"]), "H": H, "Hkv": Hkv, "D": D, "block": rng.choice([1, 2, 4, 8, 16, 32, 64])}
    if kind == "store":
        return {**c, "n_past": _log_int(rng, 1, 32000) - 1, "T": _log_int(rng, 1, 2048)}
    if kind == "load":
        return {**c, "pos0": _log_int(rng, 1, 2000) - 1, "n": _log_int(rng, 1, 16000)}
    T = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 1500)])
    n_past = _log_int(rng, 1, min(131000, 2 * 16 * 2048 * 1024 // (H * T))) - 1
    windowed = rng.random() < 0.4
    return {**c, "n_past": n_past, "T": T, "window": _log_int(rng, 1, 8192) if windowed else 0,
            "sinks": rng.choice([0, 1, 4, rng.randint(2, 150)]) if windowed else 0}


# ------------------------------------------------------------------- inputs --

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _rope_cfg(case):
    return {"n_rot": case["n_rot"], "base": 1e7, "scaling": SCALING[case["scaling"]], "factor": 4.0 if case["scaling"] != "plain" else 1.0,
            "n_ctx_orig": 32768, "beta_fast": 32.0, "beta_slow": 1.0}


def _scale(amax, kind):
    """The scale of blocks with these largest magnitudes: amax / 127 rounded to float32, or the least power of two
    with amax <= 448 of it (m 2^e with 0.5 <= m < 1: 2^(e - 9) where m <= 0.875, else 2^(e - 8))."""
    if kind == I8:
        return (amax.double() / 127).float()
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - torch.where(m <= 0.875, 9, 8)), 0)


def _code(x, s, kind):
    """The nearest codes of x / s (ties to even), as float32 code values; a scale of 0 has codes 0. The quotient
    is formed in 64 bits, so that it is on the right side of every border."""
    q = torch.where(s > 0, x.double() / torch.where(s > 0, s, 1).double(), 0)
    return q.round().float() if kind == I8 else q.float().to(torch.float8_e4m3fn).float()


def _rows(g, Hkv, n, D):
    """Keys or values [Hkv][n][D] as a layer makes them: channels of different size and mean, tokens of different size."""
    x = torch.randn(Hkv, n, D, generator=g, device=DEV)
    x *= torch.exp(0.3 * torch.randn(Hkv, 1, D, generator=g, device=DEV)) * torch.exp(0.2 * torch.randn(Hkv, n, 1, generator=g, device=DEV))
    return x + 0.5 * torch.randn(Hkv, 1, D, generator=g, device=DEV)


def _quantised(x, block, kind):
    """(codes [Hkv][N][D], scales [Hkv][N / block]) of rows padded with zeros to whole tiles of 64 positions."""
    Hkv, n, D = x.shape
    N = (n + 63) // 64 * 64
    x = torch.cat([x, x.new_zeros(Hkv, N - n, D)], 1) if N != n else x
    s = _scale(x.abs().amax(2).reshape(Hkv, N // block, block).amax(2), kind)
    c = _code(x, s.repeat_interleave(block, 1)[:, :, None], kind)
    return c.to(torch.int8 if kind == I8 else torch.float8_e4m3fn), s


def _cache(k, v, ks, vs):
    """The cache's bytes: keys [head][tile][16 positions][64 dims][4 x 16 dims][position][dim], values
    [head][tile][16 dims][4 x 4 positions][dim][16 positions][position], then the keys' and the values' scales."""
    Hkv, N, D = k.shape
    k = k.view(torch.uint8).reshape(Hkv, N // 64, 4, 16, D // 64, 4, 16).permute(0, 1, 2, 4, 5, 3, 6)
    v = v.view(torch.uint8).reshape(Hkv, N // 64, 4, 4, 4, D // 16, 16).permute(0, 1, 5, 3, 6, 2, 4)
    return torch.cat([k.reshape(-1), v.reshape(-1), ks.reshape(-1).view(torch.uint8), vs.reshape(-1).view(torch.uint8)])


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = _gen(seed)
    if case["kind"] == "rope":
        return SimpleNamespace(x=torch.randn(case["T"], case["heads"], case["D"], generator=g, device=DEV))
    H, Hkv, D, block, kind = case["H"], case["Hkv"], case["D"], case["block"], TYPE[case["type"]]
    i = SimpleNamespace(H=H, Hkv=Hkv, D=D, block=block, type=kind)
    i.n_ctx = case["pos0"] + case["n"] if case["kind"] == "load" else case["n_past"] + case["T"]
    k, v = _rows(g, Hkv, i.n_ctx, D), _rows(g, Hkv, i.n_ctx, D)
    if case["kind"] == "store":   # the cache holds the first n_past rows, the others are new, [T][Hkv * D]
        n = case["n_past"]
        i.k_new, i.v_new = (a[:, n:].transpose(0, 1).reshape(case["T"], Hkv * D).contiguous() for a in (k, v))
        k[:, n:], v[:, n:] = 0, 0
    i.k, i.ks = _quantised(k, block, kind)
    i.v, i.vs = _quantised(v, block, kind)
    if case["kind"] == "attn":
        i.qg = torch.randn(case["T"], H, 2 * D, generator=g, device=DEV)   # [query | gate] of every head
    return i


def prepare(case, seed):
    i = _inputs(case, seed)
    i.case = case
    T = case.get("T", case.get("n"))
    if case["kind"] == "rope":
        i.cfg, i.out = _rope_cfg(case), torch.empty_like(i.x)
        return i
    i.cache = _cache(i.k, i.v, i.ks, i.vs)
    if case["kind"] == "attn":
        i.out = torch.empty(T, i.H * i.D, device=DEV)
        # the program's work area for its longest chunk
        i.work = torch.zeros(1 << 28 if T > 1 else 1 << 26, dtype=torch.uint8, device=DEV)
        return i
    first, n = (case["pos0"], T) if case["kind"] == "load" else (case["n_past"] // i.block * i.block, 0)
    n = n or i.n_ctx - first
    i.first, i.n = first, n
    i.k_out, i.v_out = (torch.empty(n, i.Hkv * i.D, device=DEV) for _ in range(2))
    return i


# -------------------------------------------------------------- plain forms --

def _angles(cfg, pos0, T):
    """cos and sin [T][n_rot / 2] in 64 bits: 32 lose the angles of far positions."""
    n = cfg["n_rot"]
    f = cfg["base"] ** (-2.0 * torch.arange(n // 2, dtype=torch.float64, device=DEV) / n)
    ms = 1.0
    if cfg["scaling"] == LINEAR:
        f = f / cfg["factor"]
    if cfg["scaling"] == YARN:
        r = cfg["n_ctx_orig"] * f / (2 * math.pi)
        keep = ((r - cfg["beta_slow"]) / (cfg["beta_fast"] - cfg["beta_slow"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / cfg["factor"])
        ms = 0.1 * math.log(cfg["factor"]) + 1
    a = (pos0 + torch.arange(T, dtype=torch.float64, device=DEV))[:, None] * f
    return ms * a.cos(), ms * a.sin()


def _rotate(x, cfg, pairs, cos, sin):
    n = cfg["n_rot"]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if pairs == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., n:]], -1)


def _visible(case, j):
    """Which of the positions j each of the T rows sees, [T][len(j)]."""
    p = case["n_past"] + torch.arange(case["T"], device=DEV)[:, None]
    m = j <= p
    return m & ((j > p - case["window"]) | (j < case["sinks"])) if case["window"] else m


def _seen(case):
    """The positions that any row sees: the first tokens and the window of the chunk, or all."""
    n = case["n_past"] + case["T"]
    if not case["window"]:
        return torch.arange(n, device=DEV)
    lo = max(0, case["n_past"] - case["window"] + 1)
    s = min(case["sinks"], lo)
    return torch.cat([torch.arange(s, device=DEV), torch.arange(lo, n, device=DEV)])


def _plain_attention(i):
    case, G = i.case, i.H // i.Hkv
    T, D = case["T"], i.D
    j = _seen(case)
    if len(j) == i.k.shape[1] or not case["window"]:
        k, v, ks, vs = i.k[:, :len(j)], i.v[:, :len(j)], i.ks, i.vs
    else:
        k, v, ks, vs = (i.k.view(torch.uint8)[:, j].view(i.k.dtype), i.v.view(torch.uint8)[:, j].view(i.v.dtype), i.ks, i.vs)
    k = k.float() * ks[:, j // i.block, None]
    v = v.float() * vs[:, j // i.block, None]
    q = i.qg[..., :D].reshape(T, i.Hkv, G, D).permute(1, 0, 2, 3).reshape(i.Hkv, T * G, D)
    s = torch.matmul(q, k.transpose(1, 2)).mul_(D ** -0.5).reshape(i.Hkv, T, G, len(j))
    s.masked_fill_(~_visible(case, j)[None, :, None, :], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1)
    o = torch.matmul(s.reshape(i.Hkv, T * G, len(j)), v).reshape(i.Hkv, T, G, D) / total[..., None]
    o = o.permute(1, 0, 2, 3).reshape(T, i.H, D) / (1 + torch.exp(-i.qg[..., D:]))
    return o.reshape(T, i.H * D)


def _plain_store(i):
    """The blocks that the new rows touch after they are stored: their values [n][Hkv * D] and scales."""
    case, B = i.case, i.block
    n_old = case["n_past"] - i.first
    blocks = (i.n + B - 1) // B
    got = []
    for codes, scales, new in ((i.k, i.ks, i.k_new), (i.v, i.vs, i.v_new)):
        x = torch.zeros(i.Hkv, blocks * B, i.D, device=DEV)
        x[:, n_old:i.n] = new.reshape(-1, i.Hkv, i.D).transpose(0, 1)
        s = _scale(x.abs().amax(2).reshape(i.Hkv, blocks, B).amax(2), i.type)
        if n_old:   # a block begun earlier keeps the larger scale; its codes are rounded again where it grew
            old = scales[:, i.first // B]
            s[:, 0] = torch.maximum(s[:, 0], old)
            x[:, :n_old] = 0
        c = _code(x, s.repeat_interleave(B, 1)[:, :, None], i.type)
        if n_old:
            c[:, :n_old] = _code(codes[:, i.first:case["n_past"]].double() * old[:, None, None].double(), s[:, 0, None, None], i.type)
        y = c[:, :i.n] * s.repeat_interleave(B, 1)[:, :i.n, None]
        got.append(y.transpose(0, 1).reshape(i.n, i.Hkv * i.D))
    return {"k": got[0], "v": got[1]}


def _plain_load(i):
    j = torch.arange(i.first, i.first + i.n, device=DEV)
    return {name: (codes[:, i.first:i.first + i.n].float() * scales[:, j // i.block, None]).transpose(0, 1).reshape(i.n, i.Hkv * i.D)
            for name, codes, scales in (("k", i.k, i.ks), ("v", i.v, i.vs))}


# ------------------------------------------------------- the library's calls --

def _lib():
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "meta-work_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import xjpipe
    return xjpipe


_err = ctypes.create_string_buffer(512)


def _calls(i):
    """The pass's library calls and their arguments up to the stream, as a program keeps them, and what it returns."""
    xp, case = _lib(), i.case
    L = xp.lib()
    if case["kind"] == "rope":
        cfg = xp.XjhRopeCfg(pairs=0 if case["pairs"] == "half" else 1, **i.cfg)
        heads, D = case["heads"], case["D"]
        return i.out, [(L.xjh_rope_scaled, (i.x.data_ptr(), heads * D, D, i.out.data_ptr(), heads * D, D, case["T"], heads, D,
                                            ctypes.pointer(cfg), None, case["pos0"]))]
    c = ctypes.pointer(xp.XjhKv8(type=i.type, Hkv=i.Hkv, D=i.D, n_ctx=i.n_ctx, block=i.block, data=i.cache.data_ptr(),
                                 bytes=i.cache.numel()))
    row = i.Hkv * i.D
    if case["kind"] == "attn":
        D, q = i.D, i.qg.data_ptr()
        return i.out, [(L.xjh_attn_kv8, (c, q, i.H * 2 * D, 2 * D, q + 4 * D, i.H * 2 * D, 2 * D, case["T"], i.H, case["n_past"], None,
                                         case["window"], case["sinks"], D ** -0.5, i.out.data_ptr(), i.H * D,
                                         i.work.data_ptr(), i.work.numel()))]
    load = (L.xjh_kv8_load, (c, i.first, i.n, i.k_out.data_ptr(), row, i.v_out.data_ptr(), row))
    store = (L.xjh_kv8_store, (c, i.k_new.data_ptr(), row, i.v_new.data_ptr(), row, case["T"], case["n_past"], None)) \
        if case["kind"] == "store" else None
    return {"k": i.k_out, "v": i.v_out}, [store, load] if store else [load]


def _own(i):
    if not hasattr(i, "calls"):
        i.out, i.calls = _calls(i)
    stream = torch.cuda.current_stream().cuda_stream
    for f, args in i.calls:
        if f(*args, stream, _err, 512) != 0:
            raise RuntimeError(_err.value.decode(errors="replace"))
    return i.out


def run(i):
    if own:
        return _own(i)
    case = i.case
    if case["kind"] == "rope":
        cos, sin = _angles(i.cfg, case["pos0"], case["T"])
        return _rotate(i.x, i.cfg, case["pairs"], cos.float(), sin.float())
    return {"attn": _plain_attention, "store": _plain_store, "load": _plain_load}[case["kind"]](i)


# ------------------------------------------------------------------- bounds --

def work(case):
    if case["kind"] == "rope":
        n = case["T"] * case["heads"] * case["D"]
        return {"bytes": 8 * n, "flops": 3 * case["T"] * case["heads"] * case["n_rot"]}
    row = case["Hkv"] * case["D"]
    scales = 8 * case["Hkv"] / case["block"]   # of the keys and the values, per position
    if case["kind"] == "load":
        return {"bytes": case["n"] * (10 * row + scales), "flops": 2 * case["n"] * row}
    if case["kind"] == "store":
        T, n = case["T"], case["n_past"] % case["block"] + case["T"]
        return {"bytes": T * (10 * row + scales) + 8 * n * row, "flops": 6 * T * row}
    T, n_past, W, S = case["T"], case["n_past"], case["window"], case["sinks"]
    if W:
        lo = max(0, n_past - W + 1)
        seen = n_past + T - lo + min(S, lo)
        p = torch.arange(n_past, n_past + T, dtype=torch.int64)
        first = (p - W + 1).clamp(min=0)
        pairs = int((p + 1 - first + first.clamp(max=S)).sum())
    else:
        seen, pairs = n_past + T, T * n_past + T * (T + 1) // 2
    return {"bytes": seen * (2 * row + scales) + 12 * T * case["H"] * case["D"], "flops": 4 * pairs * case["H"] * case["D"]}


# ----------------------------------------------------------- 64-bit results --

def _exact_rope(case, x):
    n, cfg = case["n_rot"], _rope_cfg(case)
    out = x.double().clone()
    p = torch.arange(case["pos0"], case["pos0"] + case["T"], dtype=torch.float64, device=DEV)
    for i in range(n // 2):
        f, ms = cfg["base"] ** (-2.0 * i / n), 1.0
        if case["scaling"] == "linear":
            f /= cfg["factor"]
        elif case["scaling"] == "yarn":
            turns = cfg["n_ctx_orig"] * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - cfg["beta_slow"]) / (cfg["beta_fast"] - cfg["beta_slow"])))
            f, ms = f * keep + f / cfg["factor"] * (1 - keep), 0.1 * math.log(cfg["factor"]) + 1
        z = torch.polar(torch.full_like(p, ms), p * f)[:, None]
        i0, i1 = (i, i + n // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        y = torch.complex(x[:, :, i0].double(), x[:, :, i1].double()) * z
        out[:, :, i0], out[:, :, i1] = y.real, y.imag
    return out


def _exact_codes(x, s, kind):
    """Nearest code values of x / s in 64 bits, ties to even, from the formats' definitions."""
    q = x / torch.where(s > 0, s, 1.0)
    if kind == I8:
        c = torch.floor(q + 0.5)
        tie = q + 0.5 == c
        c = torch.where(tie & (c % 2 != 0), c - 1, c)
    else:   # steps of 2^(e - 3), e the exponent, at least -6
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        c = torch.round(q / step) * step
    return torch.where(s > 0, c, 0.0)


def _exact_store(case, i):
    B, kind, n0 = case["block"], TYPE[case["type"]], case["n_past"]
    first = n0 // B * B
    top = 127.0 if kind == I8 else 448.0
    out = {}
    for name, codes, scales, new in (("k", i.k, i.ks, i.k_new), ("v", i.v, i.vs, i.v_new)):
        new = new.double().reshape(case["T"], i.Hkv, i.D)
        rows = []
        for b in range(first, i.n_ctx, B):
            part = new[max(0, b - n0):b + B - n0]
            s = part.abs().amax((0, 2)) / top
            s = s.float().double() if kind == I8 else torch.where(s > 0, torch.exp2(torch.ceil(torch.log2(s.clamp(min=1e-300)))), 0.0)
            if b < n0:
                before = scales[:, b // B].double()
                s = torch.maximum(s, before)
                old = codes[:, b:n0].double().transpose(0, 1) * before[None, :, None]
                rows.append(_exact_codes(old, s[None, :, None], kind) * s[None, :, None])
            rows.append(_exact_codes(part, s[None, :, None], kind) * s[None, :, None])
        out[name] = torch.cat(rows).reshape(-1, i.Hkv * i.D)
    return out


def _exact_attention(case, i):
    T, D, G = case["T"], i.D, i.H // i.Hkv
    n = case["n_past"] + T
    j = torch.arange(n, device=DEV)
    out = torch.empty(T, i.H, D, dtype=torch.float64, device=DEV)
    for h in range(i.H):
        g = h // G
        k = i.k[g, :n].double() * i.ks[g, j // i.block, None].double()
        v = i.v[g, :n].double() * i.vs[g, j // i.block, None].double()
        for t in range(0, T, 256):
            p = case["n_past"] + torch.arange(t, min(t + 256, T), device=DEV)[:, None]
            m = (j <= p) & ((j >= p - case["window"] + 1) | (j < case["sinks"]) | (case["window"] == 0))
            s = (i.qg[t:t + 256, h, :D].double() @ k.t().contiguous()) / math.sqrt(D)
            w = torch.softmax(torch.where(m, s, -math.inf), -1)
            out[t:t + 256, h] = w @ v * torch.sigmoid(i.qg[t:t + 256, h, D:].double())
    return out.reshape(T, i.H * D)


def exact(case, seed):
    i = _inputs(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, i.x)
    if case["kind"] == "attn":
        return _exact_attention(case, i)
    if case["kind"] == "store":
        return _exact_store(case, i)
    lo, hi = case["pos0"], case["pos0"] + case["n"]
    at = torch.arange(lo, hi, device=DEV) // i.block
    return {name: (c[:, lo:hi].double() * s[:, at, None].double()).transpose(0, 1).reshape(case["n"], -1)
            for name, c, s in (("k", i.k, i.ks), ("v", i.v, i.vs))}
