// C entries of the long-context operators (the "long contexts" part of xj_hip.h):
// argument checks, the rotary frequencies, and the launches on the caller's stream.
#include "common.h"
#include "kernels.h"
#include "xj_hip.h"

#include <cmath>

using namespace xjk;

namespace {

// The stream to launch on. One of another device would run the launch there, on this device's pointers. The predefined handles
// are of the current device and no pointers, which hipStreamGetDevice takes them for.
bool stream_of(void *stream, hipStream_t &st, const char *what, char *err, size_t errlen) {
    st = (hipStream_t)stream == hipStreamLegacy ? nullptr : (hipStream_t)stream;
    if (!st || st == hipStreamPerThread) return true;
    int cur = 0;
    hipDevice_t dev = 0;
    if (hipGetDevice(&cur) != hipSuccess || hipStreamGetDevice(st, &dev) != hipSuccess) {
        (void)hipGetLastError();
        snprintf(err, errlen, "%s: not a usable stream", what);
        return false;
    }
    if ((int)dev == cur) return true;
    snprintf(err, errlen, "%s: the stream belongs to device %d, the current device is %d", what, (int)dev, cur);
    return false;
}

bool shape_ok(const xjh_kv8 *c) {
    return c && (c->type == XJH_KV_I8 || c->type == XJH_KV_E4M3) && c->Hkv >= 1 && c->Hkv <= 1024 &&
           (c->D == 64 || c->D == 128 || c->D == 256) && c->n_ctx >= 1 && c->n_ctx <= (1 << 30) && c->block >= 1 &&
           c->block <= kKvTile && (c->block & (c->block - 1)) == 0;
}

bool cache_ok(const xjh_kv8 *c, const char *what, Kv8 &out, char *err, size_t errlen) {
    if (!shape_ok(c)) {
        if (!c) snprintf(err, errlen, "%s: no cache", what);
        else
            snprintf(err, errlen, "%s: unsupported cache (type=%d, Hkv=%d, D=%d (64|128|256), n_ctx=%d, block=%d (power of two up to 64))",
                     what, c->type, c->Hkv, c->D, c->n_ctx, c->block);
        return false;
    }
    if (!c->data || ((uintptr_t)c->data & 15) || c->bytes < xjh_kv8_bytes(c)) {
        snprintf(err, errlen, "%s: the cache's memory is missing, not 16-byte aligned or below its %llu bytes", what,
                 (unsigned long long)xjh_kv8_bytes(c));
        return false;
    }
    out.e4m3 = c->type == XJH_KV_E4M3;
    out.Hkv = c->Hkv;
    out.D = c->D;
    out.n_tiles = (c->n_ctx + kKvTile - 1) / kKvTile;
    out.lg = __builtin_ctz((unsigned)c->block);
    const int64_t codes = (int64_t)c->Hkv * out.n_tiles * kKvTile * c->D;
    out.k = (uint8_t *)c->data;
    out.v = out.k + codes;
    out.ks = (float *)(out.v + codes);
    out.vs = out.ks + (((int64_t)c->Hkv * out.n_tiles * kKvTile) >> out.lg);
    return true;
}

// T tokens from n_past fit the cache.
bool range_ok(const xjh_kv8 *c, int T, int n_past, const char *what, char *err, size_t errlen) {
    if (T >= 0 && n_past >= 0 && (int64_t)n_past + T <= c->n_ctx) return true;
    snprintf(err, errlen, "%s: %d tokens at position %d do not fit %d positions", what, T, n_past, c->n_ctx);
    return false;
}

}  // namespace

extern "C" int xjh_rope_scaled(const float *x, int64_t x_tok, int64_t x_head, float *out, int64_t o_tok, int64_t o_head,
                               int T, int n_heads, int D, const xjh_rope_cfg *cfg, const int32_t *pos, int pos0,
                               void *stream, char *err, size_t errlen) {
    if (!cfg || T < 0 || n_heads < 0 || D < 2 || (int64_t)n_heads * D > (1 << 30) || cfg->n_rot < 2 || cfg->n_rot % 2 || cfg->n_rot > D ||
        cfg->n_rot / 2 > kRopeMaxPairs || (cfg->pairs != XJH_ROPE_HALF && cfg->pairs != XJH_ROPE_INTERLEAVED)) {
        snprintf(err, errlen, "rope_scaled: bad shape (T=%d, heads=%d, D=%d, n_rot=%d, pairs=%d)", T, n_heads, D,
                 cfg ? cfg->n_rot : 0, cfg ? cfg->pairs : 0);
        return -1;
    }
    const bool lin = cfg->scaling == XJH_ROPE_LINEAR, yarn = cfg->scaling == XJH_ROPE_YARN;
    if (!(cfg->base > 0.f) || !std::isfinite(cfg->base) || !std::isfinite(cfg->mscale) ||
        (!lin && !yarn && cfg->scaling != XJH_ROPE_PLAIN) || ((lin || yarn) && !(cfg->factor >= 1.f && std::isfinite(cfg->factor))) ||
        (yarn && !(cfg->n_ctx_orig > 0 && cfg->beta_fast > cfg->beta_slow && std::isfinite(cfg->beta_fast) && std::isfinite(cfg->beta_slow)))) {
        snprintf(err, errlen, "rope_scaled: bad frequencies (base=%g, scaling=%d, factor=%g, n_ctx_orig=%d, beta=%g..%g)",
                 cfg->base, cfg->scaling, cfg->factor, cfg->n_ctx_orig, cfg->beta_slow, cfg->beta_fast);
        return -1;
    }
    if (!T || !n_heads) return 0;
    if (!x || !out || (out == x && (o_tok != x_tok || o_head != x_head))) {
        snprintf(err, errlen, "rope_scaled: no buffer, or in place with other strides");
        return -1;
    }
    hipStream_t st;
    if (!stream_of(stream, st, "rope_scaled", err, errlen)) return -1;
    RopeArgs a{};
    a.x = x; a.x_tok = x_tok; a.x_head = x_head;
    a.out = out; a.o_tok = o_tok; a.o_head = o_head;
    a.T = T; a.n_heads = n_heads; a.D = D; a.n_rot = cfg->n_rot; a.interleaved = cfg->pairs == XJH_ROPE_INTERLEAVED;
    a.pos = pos; a.pos0 = pos0;
    a.mscale = cfg->mscale != 0.f ? cfg->mscale : yarn ? (float)(0.1 * std::log((double)cfg->factor) + 1.0) : 1.f;
    const double two_pi = 6.283185307179586476925;
    for (int i = 0; i < cfg->n_rot / 2; i++) {
        double f = std::pow((double)cfg->base, -2.0 * i / cfg->n_rot);
        if (lin) f /= cfg->factor;
        if (yarn) {
            double g = (cfg->n_ctx_orig * f / two_pi - cfg->beta_slow) / ((double)cfg->beta_fast - cfg->beta_slow);
            g = g < 0 ? 0 : g > 1 ? 1 : g;
            f *= g + (1 - g) / cfg->factor;
        }
        a.f[i] = f / two_pi;
    }
    if (rope_scaled_launch(a, st)) { snprintf(err, errlen, "rope_scaled launch failed"); return -1; }
    return 0;
}

extern "C" uint64_t xjh_kv8_bytes(const xjh_kv8 *c) {
    if (!shape_ok(c)) return 0;
    const uint64_t n = ((uint64_t)c->n_ctx + kKvTile - 1) / kKvTile * kKvTile;
    return 2 * (uint64_t)c->Hkv * n * c->D + 8 * (uint64_t)c->Hkv * (n / c->block);
}

extern "C" int xjh_kv8_store(const xjh_kv8 *c, const float *k, int64_t k_tok, const float *v, int64_t v_tok, int T,
                             int n_past, const int32_t *n_past_dev, void *stream, char *err, size_t errlen) {
    Kv8StoreArgs a{};
    if (!cache_ok(c, "kv8_store", a.c, err, errlen) || !range_ok(c, T, n_past, "kv8_store", err, errlen)) return -1;
    if (!T) return 0;
    if (!k || !v) { snprintf(err, errlen, "kv8_store: no rows"); return -1; }
    hipStream_t st;
    if (!stream_of(stream, st, "kv8_store", err, errlen)) return -1;
    a.k = k; a.k_tok = k_tok; a.v = v; a.v_tok = v_tok;
    a.T = T; a.npast = n_past; a.npast_dev = n_past_dev;
    if (kv8_store_launch(a, st)) { snprintf(err, errlen, "kv8_store launch failed"); return -1; }
    return 0;
}

extern "C" int xjh_kv8_load(const xjh_kv8 *c, int pos0, int n, float *k, int64_t k_tok, float *v, int64_t v_tok,
                            void *stream, char *err, size_t errlen) {
    Kv8LoadArgs a{};
    if (!cache_ok(c, "kv8_load", a.c, err, errlen) || !range_ok(c, n, pos0, "kv8_load", err, errlen)) return -1;
    if (!n || (!k && !v)) return 0;
    hipStream_t st;
    if (!stream_of(stream, st, "kv8_load", err, errlen)) return -1;
    a.k = k; a.k_tok = k_tok; a.v = v; a.v_tok = v_tok;
    a.pos0 = pos0; a.n = n;
    if (kv8_load_launch(a, st)) { snprintf(err, errlen, "kv8_load launch failed"); return -1; }
    return 0;
}

static bool attn_shape_ok(const xjh_kv8 *c, int T, int H, int n_past, int window, int n_sink) {
    return T >= 0 && H >= c->Hkv && H % c->Hkv == 0 && n_past >= 0 && (int64_t)n_past + T <= c->n_ctx && window >= 0 &&
           n_sink >= 0 && (int64_t)T * H <= (1 << 28);
}

extern "C" int xjh_attn_kv8(const xjh_kv8 *c, const float *q, int64_t q_tok, int64_t q_head, const float *gate,
                            int64_t g_tok, int64_t g_head, int T, int H, int n_past, const int32_t *n_past_dev, int window,
                            int n_sink, float scale, float *out, int64_t o_tok, void *work, size_t work_bytes, void *stream,
                            char *err, size_t errlen) {
    Kv8AttnArgs a{};
    if (!cache_ok(c, "attn_kv8", a.c, err, errlen)) return -1;
    if (!attn_shape_ok(c, T, H, n_past, window, n_sink) || !std::isfinite(scale)) {
        snprintf(err, errlen, "attn_kv8: bad shape (T=%d, H=%d on %d kv heads, n_past=%d of %d, window=%d, n_sink=%d, scale=%g)", T,
                 H, c->Hkv, n_past, c->n_ctx, window, n_sink, scale);
        return -1;
    }
    if (!T) return 0;
    if (!q || !out || ((uintptr_t)work & 15)) { snprintf(err, errlen, "attn_kv8: no buffer, or an unaligned work area"); return -1; }
    hipStream_t st;
    if (!stream_of(stream, st, "attn_kv8", err, errlen)) return -1;
    a.q = q; a.q_tok = q_tok; a.q_head = q_head;
    a.gate = gate; a.g_tok = g_tok; a.g_head = g_head;
    a.out = out; a.o_tok = o_tok;
    a.T = T; a.H = H; a.npast = n_past; a.npast_dev = n_past_dev;
    a.window = window; a.sinks = n_sink; a.scale = scale;
    a.part = (float *)work;
    if (kv8_attn_launch(a, work ? (int64_t)(work_bytes / sizeof(float)) : 0, st)) {
        snprintf(err, errlen, "attn_kv8 launch failed");
        return -1;
    }
    return 0;
}

extern "C" size_t xjh_attn_kv8_work_bytes(const xjh_kv8 *c, int T, int H, int n_past, int window, int n_sink) {
    if (!shape_ok(c) || !attn_shape_ok(c, T, H, n_past, window, n_sink) || !T) return 0;
    Kv8AttnArgs a{};
    a.c.e4m3 = c->type == XJH_KV_E4M3;
    a.c.Hkv = c->Hkv;
    a.c.D = c->D;
    a.T = T; a.H = H; a.npast = n_past; a.window = window; a.sinks = n_sink;
    return (size_t)kv8_attn_part_floats(a) * sizeof(float);
}
