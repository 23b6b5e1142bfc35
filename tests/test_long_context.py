"""The long-context entries (xjh_rope_scaled, xjh_kv8_store / _load, xjh_attn_kv8) against
plain float64 forms written here from the formulas of xj_hip.h, and what they refuse
(on the CPU, where nothing is launched).

Bars: cache codes and scales are exact (the formats define them for every input). A rotated value is
two products and a sum of values of the pair's length times a sine and cosine
of 1.5 ulp: 4 * 2^-24 of the pair's length (and of mscale). Attention: weights and queries carry 22
bits and the sums of n products are fp32, in runs of 32 keys inside an instruction: 2e-6 of
a row's largest weighted value, sum_j p_j |v_j|, holds all of it for scores up to 20 (a score s
in powers of two is off by at most 4 roundings of s: 20 * 1.44 * 4 * 2^-24 = 7e-6 in one weight and, over independent
ones, less by the root of their number; the bar for one row is 1e-5, for the norm of all rows 2e-6).
"""
import ctypes as C

import numpy as np
import pytest

import xjpipe as xp

I8, E4 = xp.KV_I8, xp.KV_E4M3
# every e4m3 value by its code
E4_VALUES = np.array([np.nan if c & 127 == 127 else (-1.0 if c & 128 else 1.0) *
                      ((c & 7) * 2.0 ** -9 if (c >> 3) & 15 == 0 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7))
                      for c in range(256)])


# ------------------------------------------------------------ plain forms --

def rope64(x, cfg, pos):
    x = x.astype(np.float64)
    n, out = cfg.n_rot, x.copy()
    i = np.arange(n // 2)
    f = float(cfg.base) ** (-2.0 * i / n)
    ms = float(cfg.mscale) or 1.0
    if cfg.scaling == xp.ROPE_LINEAR:
        f = f / cfg.factor
    if cfg.scaling == xp.ROPE_YARN:
        r = cfg.n_ctx_orig * f / (2 * np.pi)
        g = np.clip((r - cfg.beta_slow) / (float(cfg.beta_fast) - cfg.beta_slow), 0, 1)
        f = f * (g + (1 - g) / cfg.factor)
        ms = float(cfg.mscale) or 0.1 * np.log(cfg.factor) + 1
    a = np.asarray(pos, np.float64)[:, None, None] * f
    i0, i1 = (i, i + n // 2) if cfg.pairs == xp.ROPE_HALF else (2 * i, 2 * i + 1)
    u, v = x[..., i0], x[..., i1]
    out[..., i0], out[..., i1] = ms * (u * np.cos(a) - v * np.sin(a)), ms * (u * np.sin(a) + v * np.cos(a))
    return out, ms * np.hypot(u, v)


def nearest_code(x, s, kind):
    """Code values of x / s: x float64 exactly, s a float32 scale. A quotient of two 24-bit numbers is never
    within float64's rounding of a border that it is not on."""
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(s > 0, x / s, 0.0)
    q = np.where(np.isnan(x), 0.0, q)
    if kind == I8:
        return np.rint(np.clip(q, -127, 127))
    q = np.clip(q, -448, 448)
    _, e = np.frexp(q)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(q / step) * step


def block_scale(x, kind):
    m = np.abs(x.astype(np.float64))
    m = float(np.max(np.where(np.isfinite(m), m, 0.0), initial=0.0))
    if m == 0:
        return 0.0
    if kind == I8:
        return max(float(np.float32(m / 127)), 2.0 ** -126)
    s = 2.0 ** -126
    while m > 448 * s:
        s *= 2
    return s


class Ref:
    """The cache in plain arrays: code values and scales by position and block, keys and values alike."""

    def __init__(self, Hkv, D, n_ctx, block, kind):
        n = (n_ctx + 63) // 64 * 64
        self.code, self.scale = np.zeros((2, Hkv, n, D)), np.zeros((2, Hkv, n // block))
        self.Hkv, self.D, self.block, self.kind = Hkv, D, block, kind

    def store(self, k, v, n_past):
        T, B = k.shape[0], self.block
        for w, x in enumerate((k, v)):
            for g in range(self.Hkv):
                for b in range(n_past // B, (n_past + T + B - 1) // B):
                    p0, p1 = max(b * B, n_past), min(b * B + B, n_past + T)
                    rows = x[p0 - n_past:p1 - n_past, g].astype(np.float64)
                    s, old = block_scale(x[p0 - n_past:p1 - n_past, g], self.kind), self.scale[w, g, b]
                    if b * B < n_past:
                        s = max(s, old)
                        if s > old:
                            self.code[w, g, b * B:n_past] = nearest_code(self.code[w, g, b * B:n_past] * old, s, self.kind)
                    self.scale[w, g, b] = s
                    self.code[w, g, p0:p1] = nearest_code(rows, s, self.kind)

    def values(self, pos0, n):
        s = np.repeat(self.scale, self.block, 2)[:, :, pos0:pos0 + n, None]
        return (self.code[:, :, pos0:pos0 + n] * s).transpose(0, 2, 1, 3)   # [k | v][n][Hkv][D]


def unpack(cache):
    """(code values [2][Hkv][N][D], scales [2][Hkv][N / block]) of a Kv8's bytes, from the documented order."""
    c, b = cache.c, cache.bytes()
    N = (c.n_ctx + 63) // 64 * 64
    n = c.Hkv * N * c.D
    k = b[:n].reshape(c.Hkv, N // 64, 4, c.D // 64, 4, 16, 16).transpose(0, 1, 2, 5, 3, 4, 6).reshape(c.Hkv, N, c.D)
    v = b[n:2 * n].reshape(c.Hkv, N // 64, c.D // 16, 4, 16, 4, 4).transpose(0, 1, 5, 3, 6, 2, 4).reshape(c.Hkv, N, c.D)
    codes = np.stack([k, v])
    return (codes.view(np.int8).astype(np.float64) if c.type == I8 else E4_VALUES[codes],
            b[2 * n:].view(np.float32).reshape(2, c.Hkv, N // c.block))


def attend64(kv, q, n_past, gate=None, window=0, n_sink=0, scale=None):
    """kv [k | v][n][Hkv][D]. Returns (out, the rows' sum of p |v|), [T][H][D]."""
    T, H, D = q.shape
    k, v = kv.astype(np.float64)
    G, n = H // k.shape[1], k.shape[0]
    j, out, mag = np.arange(n), np.zeros((T, H, D)), np.zeros((T, H, D))
    for h in range(H):
        for t in range(T):
            p = n_past + t
            see = (j <= p) & ((window == 0) | (j > p - window) | (j < n_sink))
            s = k[see, h // G] @ q[t, h].astype(np.float64) * (D ** -0.5 if scale is None else scale)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[t, h], mag[t, h] = w @ v[see, h // G], w @ np.abs(v[see, h // G])
            if gate is not None:
                sg = 1 / (1 + np.exp(-gate[t, h].astype(np.float64)))
                out[t, h], mag[t, h] = out[t, h] * sg, mag[t, h] * sg
    return out, mag


def rows(rng, n, Hkv, D):
    """Keys or values as a layer makes them: channels and tokens of different size, channels with a mean."""
    x = rng.standard_normal((n, Hkv, D)) * np.exp(0.3 * rng.standard_normal((1, Hkv, D)) + 0.2 * rng.standard_normal((n, Hkv, 1)))
    return (x + 0.5 * rng.standard_normal((1, Hkv, D))).astype(np.float32)


# ---------------------------------------------------------------- refusals --

def _refused(name, *args):
    err = C.create_string_buffer(xp.ERR)
    rc = getattr(xp.lib(), name)(*args, err, xp.ERR)
    return rc == -1 and err.value != b""


def _cfg(**kw):
    return C.byref(xp.XjhRopeCfg(**{**dict(pairs=0, n_rot=64, base=1e4, scaling=0, factor=1.0), **kw}))


@pytest.mark.parametrize("bad", [
    dict(n_rot=63), dict(n_rot=0), dict(n_rot=-2), dict(n_rot=130), dict(pairs=2), dict(pairs=-1), dict(base=0.0), dict(base=-1.0),
    dict(base=float("nan")), dict(base=float("inf")), dict(scaling=3), dict(scaling=-1), dict(scaling=1, factor=0.5),
    dict(scaling=1, factor=float("nan")), dict(scaling=2, factor=2.0, n_ctx_orig=0, beta_fast=32, beta_slow=1),
    dict(scaling=2, factor=2.0, n_ctx_orig=4096, beta_fast=1, beta_slow=1), dict(mscale=float("inf"))])
def test_rope_refuses_bad_configurations(bad):
    assert _refused("xjh_rope_scaled", 4096, 128, 128, 8192, 128, 128, 1, 1, 128, _cfg(**bad), None, 0, None)


def test_rope_refuses_bad_shapes_and_takes_empty_ones():
    ok = (4096, 128, 128, 8192, 128, 128)
    assert _refused("xjh_rope_scaled", *ok, -1, 1, 128, _cfg(), None, 0, None)
    assert _refused("xjh_rope_scaled", *ok, 1, -1, 128, _cfg(), None, 0, None)
    assert _refused("xjh_rope_scaled", *ok, 1, 1, 32, _cfg(), None, 0, None)
    assert _refused("xjh_rope_scaled", *ok, 1, 1, 1024, _cfg(n_rot=514), None, 0, None)
    assert _refused("xjh_rope_scaled", *ok, 1, 1, 128, None, None, 0, None)
    assert _refused("xjh_rope_scaled", None, 128, 128, 8192, 128, 128, 1, 1, 128, _cfg(), None, 0, None)
    assert _refused("xjh_rope_scaled", 4096, 128, 128, None, 128, 128, 1, 1, 128, _cfg(), None, 0, None)
    assert _refused("xjh_rope_scaled", 4096, 128, 128, 4096, 256, 128, 1, 1, 128, _cfg(), None, 0, None)   # in place, moved
    err = C.create_string_buffer(xp.ERR)
    assert xp.lib().xjh_rope_scaled(None, 0, 0, None, 0, 0, 0, 4, 128, _cfg(), None, 0, None, err, xp.ERR) == 0
    assert xp.lib().xjh_rope_scaled(None, 0, 0, None, 0, 0, 4, 0, 128, _cfg(), None, 0, None, err, xp.ERR) == 0


def _kv(**kw):
    c = xp.XjhKv8(**{**dict(type=0, Hkv=2, D=128, n_ctx=100, block=32, data=4096, bytes=1 << 40), **kw})
    return C.byref(c)


BAD_CACHES = [dict(type=2), dict(type=-1), dict(Hkv=0), dict(Hkv=-1), dict(Hkv=1025), dict(D=96), dict(D=0), dict(D=512), dict(n_ctx=0),
              dict(n_ctx=-5), dict(n_ctx=(1 << 30) + 1), dict(block=0), dict(block=3), dict(block=128), dict(block=-1)]


@pytest.mark.parametrize("bad", BAD_CACHES + [dict(data=None), dict(data=4104), dict(bytes=0),
                                              dict(bytes=2 * 2 * 128 * 128 + 2 * 2 * 4 * 4 - 1)])
def test_cache_entries_refuse_bad_caches(bad):
    c = _kv(**bad)
    assert (xp.lib().xjh_kv8_bytes(c) == 0) == (bad in BAD_CACHES)
    assert _refused("xjh_kv8_store", c, 4096, 256, 4096, 256, 1, 0, None, None)
    assert _refused("xjh_kv8_load", c, 0, 1, 4096, 256, 4096, 256, None)
    assert _refused("xjh_attn_kv8", c, 4096, 256, 128, None, 0, 0, 1, 2, 0, None, 0, 0, 1.0, 4096, 256, None, 0, None)
    if bad in BAD_CACHES:
        assert xp.lib().xjh_attn_kv8_work_bytes(c, 1, 2, 0, 0, 0) == 0


def test_cache_bytes():
    # 100 positions are two tiles: 2 heads of 128 positions of 128 dims, keys and values, 4 blocks each
    assert xp.lib().xjh_kv8_bytes(_kv()) == 2 * 2 * 128 * 128 + 2 * 2 * 4 * 4
    assert xp.lib().xjh_kv8_bytes(_kv(n_ctx=1 << 30, Hkv=1024, D=256, block=1)) == 2 * 1024 * (1 << 30) * 256 + 8 * 1024 * (1 << 30)


def test_cache_entries_refuse_ranges_and_missing_rows():
    c = _kv()
    for T, n_past in ((101, 0), (1, 100), (-1, 0), (1, -1), (50, 51), ((1 << 31) - 1, (1 << 31) - 1)):
        assert _refused("xjh_kv8_store", c, 4096, 256, 4096, 256, T, n_past, None, None), (T, n_past)
        assert _refused("xjh_kv8_load", c, n_past, T, 4096, 256, 4096, 256, None), (T, n_past)
        assert _refused("xjh_attn_kv8", c, 4096, 256, 128, None, 0, 0, T, 2, n_past, None, 0, 0, 1.0, 4096, 256, None, 0, None)
        assert xp.lib().xjh_attn_kv8_work_bytes(c, T, 2, n_past, 0, 0) == 0
    assert _refused("xjh_kv8_store", c, None, 256, 4096, 256, 1, 0, None, None)
    assert _refused("xjh_kv8_store", c, 4096, 256, None, 256, 1, 0, None, None)
    assert _refused("xjh_kv8_store", None, 4096, 256, 4096, 256, 1, 0, None, None)


def test_attention_refuses_bad_arguments():
    def bad(q=4096, T=1, H=2, window=0, n_sink=0, scale=1.0, out=4096, work=None):
        return _refused("xjh_attn_kv8", _kv(), q, 256, 128, None, 0, 0, T, H, 0, None, window, n_sink, scale, out, 256, work, 0, None)
    assert bad(q=None) and bad(out=None) and bad(H=3) and bad(H=0) and bad(H=1) and bad(H=-2) and bad(window=-1) and bad(n_sink=-1)
    assert bad(scale=float("nan")) and bad(scale=float("inf")) and bad(work=4100)
    assert bad(T=100, H=1 << 30)


def test_empty_calls_do_nothing():
    err, c, L = C.create_string_buffer(xp.ERR), _kv(), xp.lib()
    assert L.xjh_kv8_store(c, None, 0, None, 0, 0, 100, None, None, err, xp.ERR) == 0
    assert L.xjh_kv8_load(c, 100, 0, None, 0, None, 0, None, err, xp.ERR) == 0
    assert L.xjh_kv8_load(c, 0, 5, None, 0, None, 0, None, err, xp.ERR) == 0
    assert L.xjh_attn_kv8(c, None, 0, 0, None, 0, 0, 0, 2, 100, None, 0, 0, 1.0, None, 0, None, 0, None, err, xp.ERR) == 0


@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("T,H,Hkv,window", [(1, 16, 4, 0), (5, 16, 4, 0), (20, 8, 1, 0), (64, 16, 4, 0), (200, 16, 4, 0), (5, 16, 4, 3000), (700, 8, 2, 0)])
def test_work_area_serves_every_earlier_position(T, H, Hkv, window, kind):
    c = _kv(type=kind, Hkv=Hkv, D=128, n_ctx=1 << 20)
    need = [xp.lib().xjh_attn_kv8_work_bytes(c, T, H, n, window, 4) for n in [*range(0, 20000, 61), 50000, 131000, 1000000]]
    assert all(a <= b for a, b in zip(need, need[1:]))


# -------------------------------------------------------------------- rope --

def _rope_close(x, cfg_kw, pos, T, **kw):
    cfg = xp.XjhRopeCfg(**cfg_kw)
    p = pos + np.arange(T) if np.isscalar(pos) else pos
    want, length = rope64(x, cfg, p)
    args = {k: v for k, v in cfg_kw.items() if k not in ("n_rot", "base", "pairs")}
    got = xp.rope_scaled(x, cfg_kw["n_rot"], cfg_kw["base"], pos, pairs=cfg_kw["pairs"], **args, **kw)
    n = cfg.n_rot
    i = np.arange(n // 2)
    i0, i1 = (i, i + n // 2) if cfg.pairs == xp.ROPE_HALF else (2 * i, 2 * i + 1)
    for e in (i0, i1):
        assert np.all(np.abs(got[..., e] - want[..., e]) <= 4 * 2.0 ** -24 * length + 1e-37)
    assert np.array_equal(got[..., n:], x[..., n:])


YARN = dict(scaling=xp.ROPE_YARN, factor=4.0, n_ctx_orig=4096, beta_fast=32.0, beta_slow=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pairs", [xp.ROPE_HALF, xp.ROPE_INTERLEAVED])
@pytest.mark.parametrize("T,H,D,n_rot,scaling,pos", [
    (1, 16, 256, 64, YARN, 100001), (5, 2, 128, 128, dict(scaling=0), 0), (3, 3, 64, 2, dict(scaling=0), (1 << 31) - 4),
    (7, 1, 96, 54, dict(scaling=xp.ROPE_LINEAR, factor=8.0), 31), (2, 8, 256, 256, {**YARN, "mscale": 0.75}, 500000),
    (300, 4, 128, 32, YARN, 4000), (2, 1, 600, 512, dict(scaling=0), 77), (4, 1, 2, 2, dict(scaling=0), 9), (1, 5, 67, 6, dict(scaling=0), 3)])
def test_rope_scaled_matches_float64(T, H, D, n_rot, scaling, pos, pairs, in_place):
    x = np.random.default_rng(T * D).standard_normal((T, H, D)).astype(np.float32)
    _rope_close(x, dict(pairs=pairs, n_rot=n_rot, base=1e6, **scaling), pos, T, in_place=in_place)


@pytest.mark.gpu
def test_rope_scaled_positions_of_its_own():
    rng = np.random.default_rng(1)
    pos = np.array([0, 7, 7, -3, 1 << 20, (1 << 31) - 1, -(1 << 31)], np.int32)
    x = rng.standard_normal((len(pos), 2, 64)).astype(np.float32)
    _rope_close(x, dict(pairs=0, n_rot=64, base=1e4, scaling=0), pos, len(pos))


@pytest.mark.gpu
def test_rope_scaled_strides_leave_the_rest_alone():
    """Queries inside rows of [query | gate] heads, 4-byte aligned, rotated in place and into another layout."""
    rng = np.random.default_rng(2)
    T, H, D, n_rot, gap = 3, 4, 64, 32, 5
    tok = H * 2 * D + gap
    buf = rng.standard_normal(T * tok + 1).astype(np.float32)
    cfg = xp.XjhRopeCfg(pairs=0, n_rot=n_rot, base=1e4, scaling=0, factor=1.0)
    x = np.stack([[buf[1 + t * tok + h * 2 * D:][:D] for h in range(H)] for t in range(T)])
    want, length = rope64(x, cfg, 9 + np.arange(T))
    dx, do, err = xp.Dev(buf), xp.Dev(np.full(T * (H * D + 3) + 1, 7, np.float32)), C.create_string_buffer(xp.ERR)
    call = xp.lib().xjh_rope_scaled
    assert call(dx.ptr + 4, tok, 2 * D, do.ptr + 4, H * D + 3, D, T, H, D, C.byref(cfg), None, 9, None, err, xp.ERR) == 0, err.value
    assert call(dx.ptr + 4, tok, 2 * D, dx.ptr + 4, tok, 2 * D, T, H, D, C.byref(cfg), None, 9, None, err, xp.ERR) == 0, err.value
    xp.lib().xjh_sync()
    o, b = do.get(np.float32, T * (H * D + 3) + 1), dx.get(np.float32, buf.shape)
    same = buf.copy()
    for t in range(T):
        y = o[1 + t * (H * D + 3):][:H * D].reshape(H, D)
        assert np.max(np.abs(y - want[t])) <= 4 * 2.0 ** -24 * length.max()
        assert np.array_equal(y[:, n_rot:], x[t][:, n_rot:])
        assert np.all(o[1 + t * (H * D + 3) + H * D:][:3] == 7)
        for h in range(H):
            same[1 + t * tok + h * 2 * D:][:n_rot] = y[h, :n_rot]
    assert o[0] == 7 and np.array_equal(b, same)


# ------------------------------------------------------------------- cache --

@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("Hkv,D,n_ctx,block,steps", [
    (1, 64, 1, 1, [1]), (2, 128, 200, 32, [1, 1, 30, 1, 63, 64, 2, 38]), (1, 256, 130, 64, [5, 60, 65]), (4, 64, 97, 1, [33, 64]),
    (3, 128, 70, 2, [1, 1, 1, 67]), (2, 256, 300, 16, [299, 1]), (1, 64, 64, 8, [3, 3, 3, 55]), (2, 64, 1000, 64, [1000])])
def test_store_codes_are_the_formats(Hkv, D, n_ctx, block, steps, kind):
    """Rows stored piece by piece (blocks begun, continued and rescaled): codes and scales equal the definition's bit for
    bit, and nothing behind the last row is touched."""
    rng = np.random.default_rng(D + n_ctx)
    cache, ref = xp.Kv8(Hkv, D, n_ctx, block, kind), Ref(Hkv, D, n_ctx, block, kind)
    cache.put_bytes(np.full(cache.c.bytes, 0xA5, np.uint8))
    before = unpack(cache)
    n = 0
    for T in steps:
        k, v = rows(rng, T, Hkv, D) * np.float32(rng.uniform(0.5, 2)), rows(rng, T, Hkv, D)
        cache.store(k, v, n)
        ref.store(k, v, n)
        n += T
        code, scale = unpack(cache)
        nb = (n + block - 1) // block
        assert np.array_equal(scale[:, :, :nb], ref.scale[:, :, :nb])
        assert np.array_equal(code[:, :, :n], ref.code[:, :, :n])
        assert np.array_equal(code[:, :, n:], before[0][:, :, n:]) and np.array_equal(scale[:, :, nb:], before[1][:, :, nb:])
    want = ref.values(0, n)
    for pos0, m in ((0, n), (n - 1, 1), (n // 3, n - n // 3)):
        k, v = cache.load(pos0, m)
        assert np.array_equal(k, want[0][pos0:pos0 + m].astype(np.float32)) and np.array_equal(v, want[1][pos0:pos0 + m].astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
def test_store_borders_and_values_that_are_not_finite(kind):
    """Every quotient on and next to a rounding border, subnormals, zeros, the largest floats, infinities and NaN."""
    D, B = 256, 4
    rng = np.random.default_rng(3)
    x = np.zeros((16, 1, D), np.float32)
    s = np.float32(0.0371)
    if kind == I8:   # block 0: borders c + 1/2 of a scale that is not a power of two, and their neighbours
        x[0, 0, 0] = np.float32(s * np.float32(127))
        b = ((np.arange(-127, 127) + 0.5) * float(np.float32(float(x[0, 0, 0]) / 127))).astype(np.float32)
        x[1, 0, :254], x[2, 0, :254], x[3, 0, :254] = b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf))
    else:
        x[0, 0, 0] = 448
        v = np.sort(E4_VALUES[np.isfinite(E4_VALUES)])
        b = ((v[1:] + v[:-1]) / 2).astype(np.float32)[:253]
        x[1, 0, :253], x[2, 0, :253], x[3, 0, :253] = b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf))
    x[4, 0] = np.float32(1e-40) * rng.standard_normal(D)             # block 1: subnormal
    x[8, 0] = rng.standard_normal(D) * np.float32(1e38)              # block 2: the largest floats
    x[8, 0, 0], x[8, 0, 1] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    x[12, 0] = rng.standard_normal(D)                                 # block 3
    x[13, 0, :4] = [np.inf, -np.inf, np.nan, 1]
    x[14, 0] = np.nan
    cache, ref = xp.Kv8(1, D, 16, B, kind), Ref(1, D, 16, B, kind)
    cache.store(x, -x, 0)
    ref.store(x, -x, 0)
    code, scale = unpack(cache)
    assert np.array_equal(scale[:, :, :4], ref.scale[:, :, :4])
    assert np.array_equal(code[:, :, :16], ref.code[:, :, :16])
    assert np.all(np.isfinite(code)) and np.all(np.isfinite(scale[:, :, :4]))


@pytest.mark.gpu
def test_store_over_older_rows_starts_its_blocks_anew():
    """Going back (a rejected draft): rows stored again over others, from the middle of a block and from its start."""
    rng = np.random.default_rng(4)
    for kind in (I8, E4):
        cache, ref = xp.Kv8(2, 64, 100, 16, kind), Ref(2, 64, 100, 16, kind)
        for n_past, T, f in ((0, 90, 4.0), (37, 20, 1.0), (48, 16, 0.25), (16, 1, 0.1)):
            k, v = rows(rng, T, 2, 64) * np.float32(f), rows(rng, T, 2, 64) * np.float32(f)
            cache.store(k, v, n_past)
            ref.store(k, v, n_past)
        code, scale = unpack(cache)
        assert np.array_equal(scale[:, :, :6], ref.scale[:, :, :6])
        assert np.array_equal(code[:, :, :90], ref.code[:, :, :90])


@pytest.mark.gpu
def test_cache_strides_and_alignment():
    """Rows inside wider ones, 4-byte aligned; loads into such, one of the two alone."""
    rng = np.random.default_rng(5)
    Hkv, D, T, tok = 2, 64, 11, 2 * 64 + 3
    k, v = (rng.standard_normal(T * tok + 1).astype(np.float32) for _ in range(2))
    cache, err, L = xp.Kv8(Hkv, D, 40, 8, I8), C.create_string_buffer(xp.ERR), xp.lib()
    dk, dv = xp.Dev(k), xp.Dev(v)
    assert L.xjh_kv8_store(C.byref(cache.c), dk.ptr + 4, tok, dv.ptr + 4, tok, T, 6, None, None, err, xp.ERR) == 0, err.value
    L.xjh_sync()
    kk, vv = (np.stack([a[1 + t * tok:][:Hkv * D].reshape(Hkv, D) for t in range(T)]) for a in (k, v))
    other = xp.Kv8(Hkv, D, 40, 8, I8)
    other.store(kk, vv, 6)
    assert np.array_equal(cache.bytes(), other.bytes())
    wk, wv = other.load(6, T)
    for which, want in ((0, wk), (1, wv)):
        d = xp.Dev(np.full(T * tok + 1, 7, np.float32))
        p = [None, None]
        p[which] = d.ptr + 4
        assert L.xjh_kv8_load(C.byref(cache.c), 6, T, p[0], tok, p[1], tok, None, err, xp.ERR) == 0, err.value
        L.xjh_sync()
        o = d.get(np.float32, T * tok + 1)
        want_o = np.full(T * tok + 1, 7, np.float32)
        for t in range(T):
            want_o[1 + t * tok:][:Hkv * D] = want[t].reshape(-1)
        assert np.array_equal(o, want_o)


# --------------------------------------------------------------- attention --

def _filled(rng, Hkv, D, n, block, kind, n_ctx=None, stale=0xFF):
    """A cache of n positions, every other byte `stale`, and its values."""
    cache = xp.Kv8(Hkv, D, n_ctx or n, block, kind)
    cache.put_bytes(np.full(cache.c.bytes, stale, np.uint8))   # 0xFF: NaN codes of e4m3, NaN scales
    cache.store(rows(rng, n, Hkv, D), rows(rng, n, Hkv, D), 0)
    return cache, np.stack(cache.load(0, n))


def _check_attn(got, want, mag, bar_row=1e-5, bar=2e-6):
    got = got.reshape(want.shape)
    assert np.all(np.isfinite(got))
    top = mag.max(-1, keepdims=True)
    assert np.max(np.abs(got - want) / top) <= bar_row
    assert np.linalg.norm((got - want) / top) <= bar * np.sqrt(want.size)


SHAPES = [  # H, Hkv, D, block, n_past, T
    (2, 1, 128, 32, 0, 1), (16, 4, 256, 32, 63, 1), (16, 4, 256, 64, 64, 1), (8, 2, 256, 16, 777, 1), (8, 8, 64, 1, 130, 1),
    (6, 2, 128, 4, 200, 1), (16, 1, 64, 64, 1000, 1), (24, 1, 128, 32, 65, 1), (16, 4, 256, 32, 1003, 5), (2, 2, 64, 8, 5, 2),
    (8, 2, 128, 2, 62, 4), (4, 4, 256, 64, 500, 33), (16, 4, 256, 32, 0, 64), (16, 2, 64, 16, 31, 100), (3, 1, 128, 1, 9, 150), (8, 2, 256, 64, 0, 257)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("H,Hkv,D,block,n_past,T", SHAPES)
def test_attention_matches_float64(H, Hkv, D, block, n_past, T, kind):
    rng = np.random.default_rng(H * D + n_past)
    n = n_past + T
    cache, kv = _filled(rng, Hkv, D, n, block, kind, n_ctx=n + 70)
    q, gate = (rng.standard_normal((T, H, D)).astype(np.float32) for _ in range(2))
    _check_attn(cache.attend(q, n_past, gate), *attend64(kv, q, n_past, gate))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (7, 4), (64, 0), (65, 64), (100, 130), (300, 2), (1 << 30, 5), (50, 1 << 30)])
@pytest.mark.parametrize("H,Hkv,D,n_past,T", [(4, 2, 128, 517, 1), (4, 1, 64, 300, 6), (8, 2, 256, 190, 70)])
def test_attention_windows_and_first_tokens(H, Hkv, D, n_past, T, window, n_sink, kind):
    rng = np.random.default_rng(window % 1000 + n_past)
    cache, kv = _filled(rng, Hkv, D, n_past + T, 16, kind)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    _check_attn(cache.attend(q, n_past, window=window, n_sink=n_sink), *attend64(kv, q, n_past, window=window, n_sink=n_sink))


@pytest.mark.gpu
@pytest.mark.parametrize("work_bytes", [0, 4, 40000, 200000, None])
def test_attention_with_less_work_area(work_bytes):
    rng = np.random.default_rng(6)
    cache, kv = _filled(rng, 2, 128, 2003, 32, I8)
    for T in (1, 3, 40):
        q = rng.standard_normal((T, 4, 128)).astype(np.float32)
        _check_attn(cache.attend(q, 2003 - T, work_bytes=work_bytes), *attend64(kv, q, 2003 - T))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
def test_attention_sharp_rising_and_equal_scores(kind):
    """Scores that reach 60 on one key, that rise from key to key (the running maximum moves in every tile) and that are
    all equal; keys and values of very different size from block to block."""
    rng = np.random.default_rng(7)
    Hkv, D, n, T = 1, 128, 700, 3
    u = rng.standard_normal(D)
    u /= np.linalg.norm(u)
    size = np.exp2(np.repeat(rng.integers(-30, 30, (n + 15) // 16), 16)[:n])[:, None, None]
    for k, v in ((np.arange(n)[:, None, None] / n * 60 * u, rows(rng, n, 1, D)),
                 (np.zeros((n, 1, D)), rows(rng, n, 1, D)),
                 (np.where(np.arange(n)[:, None, None] == 317, 60 * u, 0.1 * rng.standard_normal((n, 1, D))), rows(rng, n, 1, D)),
                 (rows(rng, n, 1, D), rows(rng, n, 1, D) * size), (np.zeros((n, 1, D)), np.zeros((n, 1, D)))):
        cache = xp.Kv8(Hkv, D, n, 16, kind)
        cache.store(k.astype(np.float32), v.astype(np.float32), 0)
        kv = np.stack(cache.load(0, n))
        q = np.tile(u.astype(np.float32), (T, 2, 1)) + (rng.standard_normal((T, 2, D)) * 0.01).astype(np.float32)
        want, mag = attend64(kv, q, n - T, scale=1.0)
        # a score of 60 is off by 4 roundings: 60 * 1.44 * 4 * 2^-24 = 2e-5 in a weight
        _check_attn(cache.attend(q, n - T, scale=1.0), want, mag + 1e-30, bar_row=4e-5, bar=2e-5)


@pytest.mark.gpu
def test_attention_of_rows_that_are_not_finite():
    """A query that is not finite stays in its own row; a key or value of a later token that was not finite
    does not reach an earlier row (the cache holds no such value)."""
    rng = np.random.default_rng(8)
    for kind in (I8, E4):
        for T in (3, 40):
            cache, kv = _filled(rng, 1, 64, 200, 1, kind)
            x = rows(rng, 1, 1, 64)
            x[0, 0, :3] = [np.inf, -np.inf, np.nan]
            cache.store(x, x, 199)
            kv = np.stack(cache.load(0, 200))
            q = rng.standard_normal((T, 4, 64)).astype(np.float32)
            q[1, 2, 5] = np.nan
            q[2, 0, 0] = np.inf
            got = cache.attend(q, 200 - T).reshape(T, 4, 64)
            q2 = np.where(np.isfinite(q), q, 0).astype(np.float32)
            want, mag = attend64(kv, q2, 200 - T)
            bad = np.zeros((T, 4), bool)
            bad[1, 2] = bad[2, 0] = True
            assert not np.any(np.isfinite(got[bad]))
            assert np.max(np.abs(got - want)[~bad] / mag.max(-1)[~bad][:, None]) < 1e-5


@pytest.mark.gpu
def test_attention_strides_alignment_and_gate():
    """Queries and gates inside [query | gate] rows with gaps, 4-byte aligned, output rows with gaps that stay."""
    rng = np.random.default_rng(9)
    for H, Hkv, D, n_past, T in ((4, 2, 64, 100, 2), (8, 2, 256, 70, 40)):
        cache, kv = _filled(rng, Hkv, D, n_past + T, 32, E4)
        tok, otok = H * 2 * D + 3, H * D + 5
        buf = rng.standard_normal(T * tok + 1).astype(np.float32)
        x = np.stack([buf[1 + t * tok:][:H * 2 * D].reshape(H, 2 * D) for t in range(T)])
        want, mag = attend64(kv, x[..., :D], n_past, x[..., D:])
        d, o, err, L = xp.Dev(buf), xp.Dev(np.full(T * otok + 1, 7, np.float32)), C.create_string_buffer(xp.ERR), xp.lib()
        wb = L.xjh_attn_kv8_work_bytes(C.byref(cache.c), T, H, n_past, 0, 0)
        work = xp.Dev(nbytes=max(wb, 16))
        assert L.xjh_attn_kv8(C.byref(cache.c), d.ptr + 4, tok, 2 * D, d.ptr + 4 + 4 * D, tok, 2 * D, T, H, n_past, None, 0, 0, D ** -0.5,
                              o.ptr + 4, otok, work.ptr, wb, None, err, xp.ERR) == 0, err.value
        L.xjh_sync()
        y = o.get(np.float32, T * otok + 1)
        got = np.stack([y[1 + t * otok:][:H * D] for t in range(T)])
        _check_attn(got, want, mag)
        rest = np.ones(T * otok + 1, bool)
        for t in range(T):
            rest[1 + t * otok:][:H * D] = False
        assert np.all(y[rest] == 7)


@pytest.mark.gpu
def test_run_together_against_the_fp16_attention():
    """Norm, rope, store, attend piece by piece over a prompt and single tokens, as a layer would, against the library's
    fp16 attention of the same projections. int8 codes with a scale per token and head are off by half a
    step of 1/127 of a row's largest value, about 3 of its deviations: the relative error of a value is
    3 / 254 / sqrt(3) = 0.7%, of keys too, and an output averages values: 3% bounds both types, whose e4m3
    codes are off by 2^-4 of the value at most and 2^-4 / sqrt(3) / 1.4 = 2.6% on the root of mean squares."""
    rng = np.random.default_rng(10)
    H, Hkv, D, n_rot, base, eps = 8, 2, 128, 64, 1e6, 1e-6
    n_ctx = 260
    qn, kn = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32), (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    qg = rng.standard_normal((n_ctx, H, 2 * D)).astype(np.float32)
    k, v = rng.standard_normal((n_ctx, Hkv, D)).astype(np.float32), rng.standard_normal((n_ctx, Hkv, D)).astype(np.float32)
    kc, vc = np.zeros((n_ctx, Hkv * D), np.uint16), np.zeros((n_ctx, Hkv * D), np.uint16)
    caches = {(kind, block): xp.Kv8(Hkv, D, n_ctx, block, kind) for kind, block in ((I8, 1), (E4, 32))}
    n = 0
    for T in (100, 33, 5, 1, 1, 64, 1):
        s = slice(n, n + T)
        want, kc, vc = xp.attn_decode(qg[s], k[s], v[s], qn, kn, kc, vc, n, n_rot, base, eps)
        q1 = xp.rope_scaled(xp.norm(qg[s, :, :D].reshape(-1, D), qn, 0, eps).reshape(T, H, D), n_rot, base, n)
        k1 = xp.rope_scaled(xp.norm(k[s].reshape(-1, D), kn, 0, eps).reshape(T, Hkv, D), n_rot, base, n)
        for key, cache in caches.items():
            cache.store(k1, v[s], n)
            got = cache.attend(q1, n, qg[s, :, D:])
            rel = np.linalg.norm(got - want) / np.linalg.norm(want)
            assert rel < 0.03 if key[0] == I8 else rel < 0.08, (key, n, T, rel)
        n += T


# ------------------------------------------- streams, graphs, sizes, positions --

def _call(name, *args):
    err = C.create_string_buffer(xp.ERR)
    assert getattr(xp.lib(), name)(*args, err, xp.ERR) == 0, err.value


class Hip:
    """Streams and graphs of the HIP runtime that the library has loaded."""

    def __init__(self):
        xp.lib()
        with open("/proc/self/maps") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        self.rt = C.CDLL(path)

    def __call__(self, name, *args):
        assert getattr(self.rt, name)(*args) == 0, name

    def stream(self):
        st = C.c_void_p()
        self("hipStreamCreate", C.byref(st))
        return st

    def capture(self, st, work):
        graph, run = C.c_void_p(), C.c_void_p()
        self("hipStreamBeginCapture", st, C.c_int(0))
        work(st)
        self("hipStreamEndCapture", st, C.byref(graph))
        self("hipGraphInstantiate", C.byref(run), graph, None, None, C.c_size_t(0))
        return run

    def sync(self):
        self("hipDeviceSynchronize")


class _Step:
    """One layer step of T tokens on a stream, position and buffers on the device: rope of queries and keys, store, attention."""

    def __init__(self, Hkv, G, D, n_ctx, block, kind, T, n_max, window=0, n_sink=0):
        self.H, self.T, self.n_max, self.window, self.n_sink = Hkv * G, T, n_max, window, n_sink
        self.cache = xp.Kv8(Hkv, D, n_ctx, block, kind)
        self.cache.put_bytes(np.full(self.cache.c.bytes, 0xFF, np.uint8))
        self.q, self.qr, self.k, self.kr, self.v, self.out = (xp.Dev(nbytes=T * h * D * 4) for h in (self.H, self.H, Hkv, Hkv, Hkv, self.H))
        self.pos, self.n_past = xp.Dev(nbytes=4 * T), xp.Dev(nbytes=4)
        self.cfg = xp.XjhRopeCfg(pairs=0, n_rot=D // 2, base=1e5, **YARN)
        self.wb = xp.lib().xjh_attn_kv8_work_bytes(C.byref(self.cache.c), T, self.H, n_max, window, n_sink)
        self.work = xp.Dev(nbytes=max(self.wb, 16))

    def run(self, st):
        c = self.cache.c
        cc, D, T, H, row = C.byref(c), c.D, self.T, self.H, c.Hkv * c.D
        for x, y, h in ((self.q, self.qr, H), (self.k, self.kr, c.Hkv)):
            _call("xjh_rope_scaled", x.ptr, h * D, D, y.ptr, h * D, D, T, h, D, C.byref(self.cfg), self.pos.ptr, 0, st)
        _call("xjh_kv8_store", cc, self.kr.ptr, row, self.v.ptr, row, T, self.n_max, self.n_past.ptr, st)
        _call("xjh_attn_kv8", cc, self.qr.ptr, H * D, D, None, 0, 0, T, H, self.n_max, self.n_past.ptr, self.window, self.n_sink, D ** -0.5,
              self.out.ptr, H * D, self.work.ptr, self.wb, st)

    def feed(self, q, k, v, n):
        for d, a in ((self.q, q), (self.k, k), (self.v, v)):
            d.put(a)
        self.n_past.put(np.array([n], np.int32))
        self.pos.put(np.arange(n, n + self.T, dtype=np.int32))

    def result(self, d=None):
        return (d or self.out).get(np.float32, (self.T, self.H, self.cache.c.D))


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,G,D,T,window,n_sink", [(2, 4, 256, 1, 0, 0), (1, 2, 128, 5, 100, 3), (2, 1, 64, 40, 0, 0),
                                                         (2, 4, 256, 200, 0, 0), (1, 4, 64, 900, 100, 70)])
def test_captured_steps_replay_at_every_position(Hkv, G, D, T, window, n_sink):
    """The four calls captured once, with the position read on the device, and replayed over a sequence with eager work and
    synchronisations between; two graphs with a cache and a work area each, on two streams at once. Every replay equals
    the eager calls bit for bit and, at the end, the float64 form."""
    rng = np.random.default_rng(D)
    hip, steps = Hip(), 9
    n_ctx = T * steps + 3
    graphs = [_Step(Hkv, G, D, n_ctx, 16, kind, T, n_ctx - T, window, n_sink) for kind in (I8, E4)]
    eager = [_Step(Hkv, G, D, n_ctx, 16, kind, T, n_ctx - T, window, n_sink) for kind in (I8, E4)]
    streams = [hip.stream() for _ in graphs]
    captured = [hip.capture(st, s.run) for s, st in zip(graphs, streams)]
    for n in range(0, T * steps, T):
        q, k, v = rng.standard_normal((T, Hkv * G, D)).astype(np.float32), rows(rng, T, Hkv, D), rows(rng, T, Hkv, D)
        for s in graphs + eager:
            s.feed(q, k, v, n)
        for g, st in zip(captured, streams):
            hip("hipGraphLaunch", g, st)
        for s in eager:
            s.run(None)
        hip.sync()
        for s, e in zip(graphs, eager):
            assert np.array_equal(s.result().view(np.uint32), e.result().view(np.uint32)), n
            assert np.array_equal(s.cache.bytes(), e.cache.bytes()), n
    for e in eager:
        kv = np.stack(e.cache.load(0, T * steps))
        _check_attn(e.result(), *attend64(kv, e.result(e.qr), T * (steps - 1), window=window, n_sink=n_sink))
    for g in captured:
        hip("hipGraphExecDestroy", g)
    for st in streams:
        hip("hipStreamDestroy", st)


@pytest.mark.gpu
def test_device_positions_outside_the_range_count_as_its_ends():
    rng = np.random.default_rng(20)
    hip = Hip()
    for given, meant in ((-5, 0), (1000, 37), (-(1 << 31), 0), ((1 << 31) - 1, 37), (20, 20)):
        a, b = (_Step(1, 2, 64, 40, 8, I8, 3, 37) for _ in range(2))
        x = [rng.standard_normal((37, 1, 64)).astype(np.float32) for _ in range(2)]
        q, k, v = (rng.standard_normal((3, h, 64)).astype(np.float32) for h in (2, 1, 1))
        for s, n in ((a, given), (b, meant)):
            s.cache.store(x[0], x[1], 0)
            s.feed(q, k, v, 0)
            s.n_past.put(np.array([n], np.int32))
            s.run(None)
        hip.sync()
        assert np.array_equal(a.result(), b.result()) and np.array_equal(a.cache.bytes(), b.cache.bytes()) and np.all(np.isfinite(a.result()))


@pytest.mark.gpu
def test_calls_follow_their_stream():
    """Work enqueued before on the caller's stream is done when the calls run: inputs that a side stream copies in behind
    half a gigabyte of other copies."""
    rng = np.random.default_rng(21)
    hip = Hip()
    s, e = (_Step(2, 2, 128, 300, 32, I8, 4, 200) for _ in range(2))
    x, q, k, v = (rng.standard_normal(n).astype(np.float32) for n in ((200, 2, 128), (4, 4, 128), (4, 2, 128), (4, 2, 128)))
    for step in (s, e):
        step.cache.store(x, x, 0)
    e.feed(q, k, v, 200)
    e.run(None)
    s.feed(q * 0, k * 0, v * 0, 200)
    src, big = [xp.Dev(y) for y in (q, k, v)], [xp.Dev(nbytes=1 << 26) for _ in range(2)]
    st = hip.stream()
    hip.sync()
    for _ in range(8):
        hip("hipMemcpyAsync", C.c_void_p(big[0].ptr), C.c_void_p(big[1].ptr), C.c_size_t(1 << 26), C.c_int(3), st)
    for d, y in zip((s.q, s.k, s.v), src):
        hip("hipMemcpyAsync", C.c_void_p(d.ptr), C.c_void_p(y.ptr), C.c_size_t(y.nbytes), C.c_int(3), st)
    s.run(st)
    hip.sync()
    hip("hipStreamDestroy", st)
    assert np.array_equal(s.result().view(np.uint32), e.result().view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
def test_cache_beyond_four_gigabytes(kind):
    """Eight heads of 256 over 2 million positions: codes past 2^32 bytes. A window's rows far into it."""
    rng = np.random.default_rng(22)
    Hkv, D, n_ctx, W = 8, 256, 1 << 21, 150
    c = xp.XjhKv8(type=kind, Hkv=Hkv, D=D, n_ctx=n_ctx, block=64)
    c.bytes = xp.lib().xjh_kv8_bytes(C.byref(c))
    assert c.bytes > 1 << 33
    buf = xp.Dev(nbytes=c.bytes)
    c.data = buf.ptr
    n, n0, T = 300, n_ctx - 300, 3
    k, v, q = rows(rng, n, Hkv, D), rows(rng, n, Hkv, D), rng.standard_normal((T, 16, D)).astype(np.float32)
    dk, dv, dq = xp.Dev(k), xp.Dev(v), xp.Dev(q)
    ok, ov, out = xp.Dev(nbytes=k.nbytes), xp.Dev(nbytes=k.nbytes), xp.Dev(nbytes=q.nbytes)
    row, cc = Hkv * D, C.byref(c)
    wb = xp.lib().xjh_attn_kv8_work_bytes(cc, T, 16, n_ctx - T, W, 0)
    work = xp.Dev(nbytes=max(wb, 16))
    _call("xjh_kv8_store", cc, dk.ptr, row, dv.ptr, row, n, n0, None, None)
    _call("xjh_kv8_load", cc, n0, n, ok.ptr, row, ov.ptr, row, None)
    _call("xjh_attn_kv8", cc, dq.ptr, 16 * D, D, None, 0, 0, T, 16, n_ctx - T, None, W, 0, D ** -0.5, out.ptr, 16 * D, work.ptr, wb, None)
    xp.lib().xjh_sync()
    shift = n0 % 64   # the same blocks at the start of a small cache
    ref = Ref(Hkv, D, n + 64, 64, kind)
    ref.store(k, v, shift)
    want = ref.values(shift, n).astype(np.float32)
    assert np.array_equal(ok.get(np.float32, k.shape), want[0]) and np.array_equal(ov.get(np.float32, k.shape), want[1])
    _check_attn(out.get(np.float32, q.shape), *attend64(want, q, n - T, window=W))
    buf.free()


@pytest.mark.gpu
def test_many_heads_and_many_rows():
    """64 kv heads (loads of more work-groups than are on the GPU at once), and a chunk of 80000 query rows checked at some."""
    rng = np.random.default_rng(23)
    cache, ref = xp.Kv8(64, 64, 700, 32, E4), Ref(64, 64, 700, 32, E4)
    k, v = rows(rng, 690, 64, 64), rows(rng, 690, 64, 64)
    cache.store(k, v, 3)
    ref.store(k, v, 3)
    want = ref.values(3, 690)
    gk, gv = cache.load(3, 690)
    assert np.array_equal(gk, want[0].astype(np.float32)) and np.array_equal(gv, want[1].astype(np.float32))
    T, H = 5000, 16
    cache, kv = _filled(rng, 2, 64, T, 64, I8)
    q = rng.standard_normal((T, H, 64)).astype(np.float32)
    got = cache.attend(q, 0).reshape(T, H, 64)
    assert np.all(np.isfinite(got))
    for t in (0, 1, 63, 64, 2500, 4999):
        _check_attn(got[t:t + 1], *attend64(kv[:, :t + 1], q[t:t + 1], t))


@pytest.mark.gpu
@pytest.mark.parametrize("T,n_past", [(1, 3000), (3, 3000), (40, 3000), (300, 0), (9, 20000), (300, 3000)])
def test_the_same_call_gives_the_same_bits(T, n_past):
    rng = np.random.default_rng(24)
    cache, _ = _filled(rng, 4, 128, n_past + T, 32, I8)
    q = rng.standard_normal((T, 8, 128)).astype(np.float32)
    a = cache.attend(q, n_past)
    for _ in range(3):
        assert np.array_equal(a.view(np.uint32), cache.attend(q, n_past).view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_attention_scales_of_any_sign(scale):
    rng = np.random.default_rng(25)
    for T, n_past in ((1, 200), (60, 70)):
        for kind in (I8, E4):
            cache, kv = _filled(rng, 1, 64, n_past + T, 32, kind)
            q = rng.standard_normal((T, 2, 64)).astype(np.float32)
            _check_attn(cache.attend(q, n_past, scale=scale, window=90, n_sink=2),
                        *attend64(kv, q, n_past, scale=scale, window=90, n_sink=2))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("T,H", [(1, 4), (2, 4), (4, 4), (9, 4), (50, 2)])   # 4, 8, 16 rows a work-group and more
@pytest.mark.parametrize("window,n_sink,n_past", [(100, 4, 700), (70, 0, 300), (1, 70, 200), (65, 64, 129)])
def test_attention_of_positions_that_were_never_stored(window, n_sink, n_past, T, H, kind):
    """Only the first tokens and the window's are in the cache; every other byte is a NaN code or scale."""
    rng = np.random.default_rng(26)
    D, n = 64, n_past + T
    lo = n_past - window + 1
    k, v = rows(rng, n, 2, D), rows(rng, n, 2, D)
    cache, ref = xp.Kv8(2, D, n + 80, 1, kind), Ref(2, D, n + 80, 1, kind)
    cache.put_bytes(np.full(cache.c.bytes, 0xFF, np.uint8))
    for p0, p1 in ((0, n_sink), (lo, n)):
        cache.store(k[p0:p1], v[p0:p1], p0)
        ref.store(k[p0:p1], v[p0:p1], p0)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    _check_attn(cache.attend(q, n_past, window=window, n_sink=n_sink),
                *attend64(ref.values(0, n), q, n_past, window=window, n_sink=n_sink))


@pytest.mark.gpu
def test_rope_scaled_of_very_many_tokens():
    """2^24 + 3 tokens, two elements each: more work-groups than one dimension of a grid takes."""
    T, D = (1 << 24) + 3, 2
    cfg = xp.XjhRopeCfg(pairs=0, n_rot=2, base=1e4, scaling=0, factor=1.0)
    x = np.random.default_rng(27).standard_normal((T, 1, D)).astype(np.float32)
    got = xp.rope_scaled(x, 2, 1e4, 5)
    for t0 in (0, (1 << 23) - 2, (1 << 24) - 2):
        want, length = rope64(x[t0:t0 + 5], cfg, 5 + t0 + np.arange(5))
        assert np.all(np.abs(got[t0:t0 + 5] - want) <= 4 * 2.0 ** -24 * length[..., :1] + 1e-37)


@pytest.mark.gpu
def test_wrappers_refuse_arrays_of_other_shapes_and_take_empty_ones():
    rng = np.random.default_rng(28)
    cache = xp.Kv8(2, 64, 100)
    x = rows(rng, 5, 2, 64)
    for call in (lambda: cache.store(x, x[:4], 0), lambda: cache.store(x[:, :1], x[:, :1], 0), lambda: cache.store(x[..., :32], x[..., :32], 0),
                 lambda: cache.attend(np.zeros((1, 2, 128)), 0), lambda: cache.attend(x, 0, gate=x[:3]), lambda: cache.attend(x[0], 0),
                 lambda: xp.rope_scaled(x, 64, 1e4, np.zeros(4, np.int32)), lambda: xp.rope_scaled(x[0], 64, 1e4, 0)):
        with pytest.raises(xp.XjError):
            call()
    assert not np.any(cache.bytes())
    cache.store(x[:0], x[:0], 100)
    assert not np.any(cache.bytes())
    assert cache.attend(x[:0], 100).shape == (0, 128) and xp.rope_scaled(x[:0], 64, 1e4, 0).shape == (0, 2, 64)
    assert cache.load(100, 0)[0].shape == (0, 2, 64)


# Enough rows and tiles for the kernel that takes 32 rows at a time (fewer go to the one that takes 8 or 16).

@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("H,Hkv,D,block,n_past,T", [(8, 2, 256, 32, 400, 300), (8, 2, 128, 1, 390, 301), (16, 4, 64, 64, 411, 170), (3, 1, 256, 16, 1200, 299),
                                                         (8, 2, 256, 32, 300, 700), (8, 2, 128, 1, 300, 500), (16, 4, 256, 64, 0, 512)])
def test_attention_of_many_rows_matches_float64(H, Hkv, D, block, n_past, T, kind):
    rng = np.random.default_rng(H * D + n_past)
    n = n_past + T
    cache, kv = _filled(rng, Hkv, D, n, block, kind, n_ctx=n + 70)
    q, gate = (rng.standard_normal((T, H, D)).astype(np.float32) for _ in range(2))
    _check_attn(cache.attend(q, n_past, gate), *attend64(kv, q, n_past, gate))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (7, 4), (65, 64), (100, 130), (300, 2), (200, 0), (100, 4)])
def test_windows_of_many_rows(window, n_sink, kind):
    """Of the positions before the call only the first tokens and the window's are stored, the other bytes are NaN codes and scales."""
    rng = np.random.default_rng(30)
    T, H, D, n_past = 700, 8, 64, 430
    n, lo = n_past + T, n_past - window + 1
    k, v = rows(rng, n, 2, D), rows(rng, n, 2, D)
    cache, ref = xp.Kv8(2, D, n + 80, 1, kind), Ref(2, D, n + 80, 1, kind)
    cache.put_bytes(np.full(cache.c.bytes, 0xFF, np.uint8))
    for p0, p1 in ((0, n_sink), (lo, n)):
        cache.store(k[p0:p1], v[p0:p1], p0)
        ref.store(k[p0:p1], v[p0:p1], p0)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    _check_attn(cache.attend(q, n_past, window=window, n_sink=n_sink),
                *attend64(ref.values(0, n), q, n_past, window=window, n_sink=n_sink))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("work_bytes", [0, 200000, None])
def test_split_rows_of_a_long_context(work_bytes, kind):
    rng = np.random.default_rng(31)
    T, n = 9, 20009
    cache, kv = _filled(rng, 4, 64, n, 32, kind)
    q = rng.standard_normal((T, 16, 64)).astype(np.float32)
    _check_attn(cache.attend(q, n - T, work_bytes=work_bytes), *attend64(kv, q, n - T))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
def test_many_rows_of_sharp_scores_and_rows_that_are_not_finite(kind):
    """Scores that rise to 60 from key to key, or reach it on one key; a query that is not finite stays in its own row."""
    rng = np.random.default_rng(32)
    D, n, T, H = 128, 1500, 500, 4
    u = rng.standard_normal(D)
    u /= np.linalg.norm(u)
    for k in (np.arange(n)[:, None, None] / n * 60 * u, np.where(np.arange(n)[:, None, None] == 317, 60 * u, 0.1 * rng.standard_normal((n, 1, D)))):
        cache = xp.Kv8(1, D, n, 16, kind)
        cache.store(k.astype(np.float32), rows(rng, n, 1, D), 0)
        kv = np.stack(cache.load(0, n))
        q = np.tile(u.astype(np.float32), (T, H, 1)) + (rng.standard_normal((T, H, D)) * 0.01).astype(np.float32)
        want, mag = attend64(kv, q, n - T, scale=1.0)
        # a score of 60 is off by 4 roundings: 60 * 1.44 * 4 * 2^-24 = 2e-5 in a weight
        _check_attn(cache.attend(q, n - T, scale=1.0), want, mag + 1e-30, bar_row=4e-5, bar=2e-5)
        q[5, 1, 7], q[250, 3, 0], q[299, 0, 127] = np.nan, np.inf, -np.inf
        bad = ~np.isfinite(q).all(-1)
        got = cache.attend(q, n - T, scale=1.0).reshape(q.shape)
        assert not np.any(np.isfinite(got[bad])) and bad.sum() == 3
        assert np.max(np.abs(got - want)[~bad] / (mag.max(-1)[~bad][:, None] + 1e-30)) <= 4e-5


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("T,H,Hkv,D,n_past,window,n_sink", [(1, 4, 2, 128, 330, 0, 0), (1, 8, 1, 64, 447, 0, 0), (3, 4, 1, 128, 1000, 0, 0), (4, 8, 2, 64, 800, 0, 0),
                                                            (1, 4, 2, 64, 1500, 500, 70), (4, 4, 1, 128, 1501, 500, 70), (12, 1, 1, 64, 378, 0, 0)])
def test_unsplit_rows_of_many_tiles(T, H, Hkv, D, n_past, window, n_sink, kind):
    """Work-groups of 6, 7, 8 and more tiles one after the other (no work area), the last one whole, begun or half in a window."""
    rng = np.random.default_rng(n_past)
    cache, kv = _filled(rng, Hkv, D, n_past + T, 8, kind, n_ctx=n_past + T + 64)
    q, gate = (rng.standard_normal((T, H, D)).astype(np.float32) for _ in range(2))
    _check_attn(cache.attend(q, n_past, gate, window=window, n_sink=n_sink, work_bytes=0),
                *attend64(kv, q, n_past, gate, window=window, n_sink=n_sink))


@pytest.mark.gpu
def test_store_borders_at_the_smallest_scales():
    """int8 scales in [2^-126, 2^-125), half of which is no float when their last bit is odd: quotients on and next to every border."""
    B, D = 4, 256
    u = np.float32(2.0 ** -126)
    tops = [np.float32(127 * (float(u) + i * 2.0 ** -149)) for i in (1, 2, 1025, 3333333, 4194303, 4194305, 7340033, 8388607)] + [np.float32(1.754825e-36)]
    x = np.zeros((B * len(tops), 1, D), np.float32)
    for i, top in enumerate(tops):
        s = float(np.float32(float(top) / 127))
        b = ((np.arange(-127, 127) + 0.5) * s).astype(np.float32)
        x[B * i, 0, 0] = top
        for j, y in enumerate((b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf)))):
            x[B * i + 1 + j, 0, :254] = np.clip(y, -top, top)
    cache, ref = xp.Kv8(1, D, len(x), B, I8), Ref(1, D, len(x), B, I8)
    cache.store(x, -x, 0)
    ref.store(x, -x, 0)
    code, scale = unpack(cache)
    n = len(tops)
    assert np.all(ref.scale[:, :, :n] >= 2.0 ** -126) and np.all(ref.scale[:, :, :n] <= 2.0 ** -125)
    assert np.array_equal(scale[:, :, :n], ref.scale[:, :, :n])
    assert np.array_equal(code[:, :, :len(x)], ref.code[:, :, :len(x)])


# (rows of 8, of 16 and of 32 a work-group)
ROWS = [(3, 2, 700), (4, 4, 700), (200, 8, 1300)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,n", ROWS)
@pytest.mark.parametrize("kind", [I8, E4])
def test_attention_of_the_largest_values(kind, T, H, n):
    """Value blocks whose scale times 128 is no float any more (int8), equal scores."""
    rng = np.random.default_rng(39)
    D = 64
    v = rows(rng, n, 1, D).astype(np.float64)
    for b in range(0, n, 16):
        v[b:b + 16] *= float(np.finfo(np.float32).max) * (0.995 if kind == I8 else 0.9) / np.abs(v[b:b + 16]).max()
    v = v.astype(np.float32)
    cache, ref = xp.Kv8(1, D, n, 16, kind), Ref(1, D, n, 16, kind)
    cache.store(v * 0, v, 0)
    ref.store(v * 0, v, 0)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    for work_bytes in (0, None):
        _check_attn(cache.attend(q, n - T, work_bytes=work_bytes), *attend64(ref.values(0, n), q, n - T))


def _sized(rng, sizes, n, D, kind):
    """n positions whose blocks of 16 values have the largest magnitudes `sizes` in turn: the cache and its values in float64."""
    k, v = rows(rng, n, 1, D), rows(rng, n, 1, D).astype(np.float64)
    for b in range(0, n, 16):
        v[b:b + 16] *= sizes[b // 16 % len(sizes)] / np.abs(v[b:b + 16]).max()
    v = v.astype(np.float32)
    cache, ref = xp.Kv8(1, D, n, 16, kind), Ref(1, D, n, 16, kind)
    cache.store(k, v, 0)
    ref.store(k, v, 0)
    return cache, ref.values(0, n)


@pytest.mark.gpu
@pytest.mark.parametrize("work_bytes", [0, None])
@pytest.mark.parametrize("T,H,n", ROWS)
@pytest.mark.parametrize("kind", [I8, E4])
def test_attention_of_values_of_any_size(kind, T, H, n, work_bytes):
    """Value blocks of very different size, up to the largest floats (those whose codes' values are still floats): everywhere, first, in the
    middle, last, beside zeros. The small ones count in the total as much as the large ones. Bars as for any size: totals and
    sums are rounded relative to themselves."""
    rng = np.random.default_rng(40)
    top = float(np.finfo(np.float32).max) * (0.995 if kind == I8 else 0.9)
    q = rng.standard_normal((T, H, 64)).astype(np.float32)
    blocks = n // 16 + 1
    for sizes in (np.exp2(rng.integers(-30, 30, blocks)), [top], [1e37], [1e32, 1e-3],
                  [top] + [1.0] * (blocks - 1), [1.0] * (blocks // 2) + [top] + [1.0] * blocks, [1e-6] * (blocks - 2) + [top] * 2, [1e-30], [0.0, 1e-6]):
        cache, kv = _sized(rng, sizes, n, 64, kind)
        want, mag = attend64(kv, q, n - T)
        _check_attn(cache.attend(q, n - T, work_bytes=work_bytes), want, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,n", ROWS)
@pytest.mark.parametrize("ratio,D", [(4, 64), (16, 128), (100, 256), (1000, 64)])
@pytest.mark.parametrize("kind", [I8, E4])
def test_attention_of_queries_with_a_large_channel(kind, ratio, D, T, H, n):
    """Queries with one channel `ratio` times the others, keys that are small in it, so that every channel moves the scores alike. A query
    element is off by 2^-22 of itself or by 2^-30 of its row's largest, about 4 `ratio`: 4e-6 at 1000, a third of which, on the root of mean squares,
    enters a score of D channels over the root of D, so 1.3e-6 of a weight and, over hundreds of independent weights, less than the bars of any query."""
    rng = np.random.default_rng(41)
    c = 11
    k, v = rows(rng, n, 1, D), rows(rng, n, 1, D)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    k[..., c] /= ratio
    q[..., c] *= ratio
    # a block's scale is its largest element's: the small channel's keys are few codes, which the float64 form takes as they are
    cache = xp.Kv8(1, D, n, 1, kind)
    cache.store(k, v, 0)
    kv = np.stack(cache.load(0, n))
    _check_attn(cache.attend(q, n - T), *attend64(kv, q, n - T))


@pytest.mark.parametrize("n_heads,D", [((1 << 31) - 1, 2), ((1 << 23) + 1, 128), (1, (1 << 30) + 1), (1 << 20, 1 << 20)])
def test_rope_refuses_tokens_of_more_elements_than_a_work_group_counts(n_heads, D):
    """n_heads * D above 2^30: the kernel's index of a token's elements would pass 31 bits."""
    err = C.create_string_buffer(xp.ERR)
    for T in (0, 1):
        assert xp.lib().xjh_rope_scaled(4096, D, D, 4096, D, D, T, n_heads, D, _cfg(n_rot=2), None, 0, None, err, xp.ERR) == -1
        assert b"bad shape" in err.value
    assert xp.lib().xjh_rope_scaled(4096, 128, 128, 4096, 128, 128, 0, 1 << 23, 128, _cfg(n_rot=2), None, 0, None, err, xp.ERR) == 0


@pytest.mark.gpu
def test_cache_beyond_four_gigabytes_of_cleared_memory():
    """As test_cache_beyond_four_gigabytes, with the begun block's bytes and scale cleared first, as the store asks for."""
    rng = np.random.default_rng(42)
    hip, Hkv, D, n_ctx = Hip(), 8, 256, 1 << 21
    for kind in (I8, E4):
        c = xp.XjhKv8(type=kind, Hkv=Hkv, D=D, n_ctx=n_ctx, block=64)
        c.bytes = xp.lib().xjh_kv8_bytes(C.byref(c))
        assert c.bytes > 1 << 33
        buf = xp.Dev(nbytes=c.bytes)
        c.data = buf.ptr
        hip("hipMemset", C.c_void_p(buf.ptr), C.c_int(0), C.c_size_t(c.bytes))
        n, n0 = 300, n_ctx - 300
        k, v = rows(rng, n, Hkv, D), rows(rng, n, Hkv, D)
        dk, dv, ok, ov = xp.Dev(k), xp.Dev(v), xp.Dev(nbytes=k.nbytes), xp.Dev(nbytes=v.nbytes)
        row, cc = Hkv * D, C.byref(c)
        _call("xjh_kv8_store", cc, dk.ptr, row, dv.ptr, row, n, n0, None, None)
        _call("xjh_kv8_load", cc, n0, n, ok.ptr, row, ov.ptr, row, None)
        xp.lib().xjh_sync()
        ref = Ref(Hkv, D, n + 64, 64, kind)
        ref.store(k, v, n0 % 64)
        want = ref.values(n0 % 64, n).astype(np.float32)
        assert np.array_equal(ok.get(np.float32, k.shape), want[0]) and np.array_equal(ov.get(np.float32, k.shape), want[1])
        buf.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("Hkv,G,D,T,window,n_sink", [(2, 4, 64, 1, 0, 0), (1, 4, 128, 5, 0, 0), (1, 4, 64, 40, 0, 0), (1, 4, 64, 5, 1000, 70)])
def test_captured_step_far_below_its_bound(Hkv, G, D, T, window, n_sink, kind):
    """A step captured with a bound of 60000 positions and replayed at a few hundred and a few thousand, from the first on."""
    rng = np.random.default_rng(43)
    hip, n_max = Hip(), 60000
    s = _Step(Hkv, G, D, n_max + T, 32, kind, T, n_max, window, n_sink)
    st = hip.stream()
    g = hip.capture(st, s.run)
    n = 0
    for gap in (0, 3, 190, 1, 2100, 2500):
        if gap:
            s.cache.store(rows(rng, gap, Hkv, D), rows(rng, gap, Hkv, D), n)
            n += gap
        s.feed(rng.standard_normal((T, Hkv * G, D)).astype(np.float32), rows(rng, T, Hkv, D), rows(rng, T, Hkv, D), n)
        hip.sync()
        for _ in range(2):
            hip("hipGraphLaunch", g, st)
        hip.sync()
        kv = np.stack(s.cache.load(0, n + T))
        _check_attn(s.result(), *attend64(kv, s.result(s.qr), n, window=window, n_sink=n_sink))
        n += T
    hip("hipGraphExecDestroy", g)
    hip("hipStreamDestroy", st)


@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H,Hkv,window", [(1, 16, 4, 0), (1, 8, 2, 0), (1, 2, 1, 0), (2, 16, 16, 0), (5, 16, 4, 0), (33, 16, 4, 0), (64, 32, 8, 0),
                                            (300, 16, 4, 0), (340, 16, 4, 0), (5, 16, 4, 3000), (700, 8, 2, 2000)])
def test_work_area_serves_every_earlier_position_of_any_dims(T, H, Hkv, window, D, kind):
    """The splits' rules differ by dims and heads: the area asked for is never less at a later position."""
    c = _kv(type=kind, Hkv=Hkv, D=D, n_ctx=1 << 20)
    need = [xp.lib().xjh_attn_kv8_work_bytes(c, T, H, n, window, 4) for n in [*range(0, 20000, 61), 24000, 30000, 50000, 131000, 1000000]]
    assert all(a <= b for a, b in zip(need, need[1:]))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,n", ROWS)
@pytest.mark.parametrize("kind", [I8, E4])
def test_attention_of_keys_of_any_size(kind, T, H, n):
    """Keys up to 1e37: of queries as small as they are large, and of others, whose scores of 1e6 to 1e37 leave one key a row."""
    rng = np.random.default_rng(44)
    D = 64
    k, v, q = rows(rng, n, 1, D), rows(rng, n, 1, D), rng.standard_normal((T, H, D)).astype(np.float32)
    for fk, fq in ((1e34, 1e-34), (1e30, 1e-30), (1e-28, 1e28), (1e6, 1.0), (3.0, 3e8), (1e4, 1e7), (1e34, 1.0), (3e36, 1.0), (1.0, 1e36)):
        cache, ref = xp.Kv8(1, D, n, 16, kind), Ref(1, D, n, 16, kind)
        kf, qf = k * np.float32(fk), q * np.float32(fq)
        cache.store(kf, v, 0)
        ref.store(kf, v, 0)
        _check_attn(cache.attend(qf, n - T), *attend64(ref.values(0, n), qf, n - T))


@pytest.mark.gpu
@pytest.mark.parametrize("handle", [1, 2])
def test_predefined_stream_handles(handle):
    """hipStreamLegacy and hipStreamPerThread, small numbers instead of pointers: a layer step on each gives the default stream's bits."""
    rng = np.random.default_rng(45)
    a, b = (_Step(2, 2, 64, 200, 16, I8, 3, 100) for _ in range(2))
    x = rng.standard_normal((100, 2, 64)).astype(np.float32)
    q, k, v = (rng.standard_normal((3, h, 64)).astype(np.float32) for h in (4, 2, 2))
    for s, stream in ((a, handle), (b, None)):
        s.cache.store(x, x, 0)
        s.feed(q, k, v, 100)
        s.run(stream)
        xp.lib().xjh_sync()
    assert np.array_equal(a.result().view(np.uint32), b.result().view(np.uint32)) and np.array_equal(a.cache.bytes(), b.cache.bytes())
    out = xp.Dev(nbytes=3 * 2 * 64 * 4)
    _call("xjh_kv8_load", C.byref(a.cache.c), 100, 3, out.ptr, 128, None, 0, handle)
    xp.lib().xjh_sync()
    assert np.array_equal(out.get(np.float32, (3, 2, 64)), a.cache.load(100, 3)[0])


def test_wrappers_refuse_numbers_that_are_no_int32():
    """ctypes cuts them: position 2^32 would be 0."""
    x = np.zeros((2, 2, 64), np.float32)
    cache = xp.Kv8.__new__(xp.Kv8)   # (without memory: nothing is launched)
    cache.c = xp.XjhKv8(type=I8, Hkv=2, D=64, n_ctx=100, block=8)
    for call in (lambda: xp.rope_scaled(x, 64, 1e4, 1 << 31), lambda: xp.rope_scaled(x, 64, 1e4, np.array([0, 1 << 32])),
                 lambda: xp.rope_scaled(x, 64, 1e4, [0, -(1 << 31) - 1]), lambda: cache.store(x, x, 1 << 32), lambda: cache.load(1 << 32, 1),
                 lambda: cache.load(0, 1 << 32), lambda: cache.attend(x, 1 << 32), lambda: cache.attend(x, 5, window=1 << 32),
                 lambda: cache.attend(x, 5, n_sink=1 << 32), lambda: xp.Kv8(2, 64, (1 << 32) + 1), lambda: xp.Kv8((1 << 32) + 2, 64, 1)):
        with pytest.raises(xp.XjError, match="int32"):
            call()
