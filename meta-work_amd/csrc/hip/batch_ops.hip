// C entries of the operators for several requests (the "several requests" part of xj_hip.h): argument checks
// and the launches on the caller's stream.
#include "common.h"
#include "kernels.h"
#include "xj_hip.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>

using namespace xjk;

namespace {

bool page_ok(int page, int n_pages) {
    return page >= 16 && page <= 256 && (page & (page - 1)) == 0 && n_pages >= 1 && (int64_t)n_pages * page <= INT32_MAX;
}

bool shape_ok(const xjh_paged *c) {
    return c && (c->type == XJ_F16 || c->type == XJ_BF16) && c->Hkv >= 1 && c->Hkv <= 1024 &&
           (c->D == 64 || c->D == 128 || c->D == 256) && page_ok(c->page, c->n_pages);
}

bool cache_ok(const xjh_paged *c, const char *what, Paged &out, char *err, size_t errlen) {
    if (!shape_ok(c)) {
        if (!c) snprintf(err, errlen, "%s: no cache", what);
        else
            snprintf(err, errlen, "%s: unsupported cache (type=%d (f16|bf16), Hkv=%d, D=%d (64|128|256), page=%d (16|32|64|128|256), n_pages=%d)",
                     what, c->type, c->Hkv, c->D, c->page, c->n_pages);
        return false;
    }
    if (!c->k || !c->v || (((uintptr_t)c->k | (uintptr_t)c->v) & 15) || c->bytes < xjh_paged_bytes(c)) {
        snprintf(err, errlen, "%s: the cache's memory is missing, not 16-byte aligned or below its %llu bytes", what,
                 (unsigned long long)xjh_paged_bytes(c));
        return false;
    }
    out.k = c->k;
    out.v = c->v;
    out.bf16 = c->type == XJ_BF16;
    out.Hkv = c->Hkv;
    out.D = c->D;
    out.lg = __builtin_ctz((unsigned)c->page);
    out.n_pages = c->n_pages;
    return true;
}

int row_type(int type) { return type == XJ_F32 ? kRowF32 : type == XJ_F16 ? kRowF16 : type == XJ_BF16 ? kRowBf16 : -1; }

constexpr int kMaxReq = 65536;

struct Span {
    const void *p;
    uint64_t bytes;
};
bool overlap(Span x, Span y) {
    const uint64_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
    return a && b && a < b + y.bytes && b < a + x.bytes;
}

}  // namespace

extern "C" size_t xjh_page_plan_work_bytes(int n_req) {
    return n_req < 0 || n_req > kMaxReq ? 0 : (2 * ((size_t)n_req + 1) + 4) * sizeof(int32_t);
}

extern "C" int xjh_page_plan(const xjh_pages *p, const int32_t *held, const int32_t *n_past, const int32_t *n_new, int n_req,
                             const int32_t *n_free, int32_t *n_free_out, int T, int32_t *cu, int32_t *kv_len, int32_t *pos,
                             int32_t *slot, int32_t *status, void *work, size_t work_bytes, void *stream, char *err,
                             size_t errlen) {
    if (!p || !page_ok(p->page, p->n_pages) || p->max_blocks < 1 || (int64_t)p->max_blocks * p->page > INT32_MAX || n_req < 0 ||
        n_req > kMaxReq || (int64_t)n_req * p->max_blocks > (1 << 30) || T < 0) {
        snprintf(err, errlen, "page_plan: bad shape (page=%d (16|32|64|128|256), n_pages=%d, max_blocks=%d, n_req=%d, T=%d)",
                 p ? p->page : 0, p ? p->n_pages : 0, p ? p->max_blocks : 0, n_req, T);
        return -1;
    }
    if (!p->free_list || !n_free || !n_free_out || !cu || !status || (n_req && (!p->table || !n_past || !n_new || !kv_len))) {
        snprintf(err, errlen, "page_plan: a buffer is missing");
        return -1;
    }
    if (!work || ((uintptr_t)work & 15) || work_bytes < xjh_page_plan_work_bytes(n_req)) {
        snprintf(err, errlen, "page_plan: the work area is missing, not 16-byte aligned or below its %llu bytes",
                 (unsigned long long)xjh_page_plan_work_bytes(n_req));
        return -1;
    }
    // the lengths are read again after the first results are written
    const uint64_t row = 4 * (uint64_t)n_req, rows = 4 * (uint64_t)T;
    for (const Span in : {Span{held, row}, Span{n_past, row}, Span{n_new, row}})
        for (const Span to : {Span{n_free_out, 4}, Span{cu, row + 4}, Span{kv_len, row}, Span{pos, rows}, Span{slot, rows}, Span{status, 16},
                              Span{work, work_bytes}, Span{p->table, row * p->max_blocks}, Span{p->free_list, 4 * (uint64_t)p->n_pages}})
            if (overlap(in, to)) {
                snprintf(err, errlen, "page_plan: the requests' lengths lie in a buffer that is written");
                return -1;
            }
    hipStream_t st;
    if (!stream_of(stream, st, "page_plan", err, errlen)) return -1;
    PlanArgs a{};
    a.lg = __builtin_ctz((unsigned)p->page);
    a.n_pages = p->n_pages; a.max_blocks = p->max_blocks;
    a.table = p->table; a.free_list = p->free_list;
    a.held = held; a.n_past = n_past; a.n_new = n_new;
    a.n_req = n_req; a.T = T;
    a.n_free = n_free; a.n_free_out = n_free_out;
    a.cu = cu; a.kv_len = kv_len; a.pos = pos; a.slot = slot; a.status = status;
    a.sum = (int32_t *)work;
    a.rel_cu = a.sum + 4;
    a.take_cu = a.rel_cu + n_req + 1;
    if (page_plan_launch(a, st)) { snprintf(err, errlen, "page_plan launch failed"); return -1; }
    return 0;
}

extern "C" uint64_t xjh_paged_bytes(const xjh_paged *c) {
    return shape_ok(c) ? 2 * (uint64_t)c->n_pages * c->page * c->Hkv * c->D : 0;
}

extern "C" int xjh_paged_store(const xjh_paged *c, int type, const void *k, int64_t k_tok, const void *v, int64_t v_tok, int T,
                               const int32_t *slot, void *stream, char *err, size_t errlen) {
    PagedStoreArgs a{};
    if (!cache_ok(c, "paged_store", a.c, err, errlen)) return -1;
    if (T < 0 || (int64_t)T * c->Hkv > (1 << 26) || (type != XJ_F32 && type != c->type)) {
        snprintf(err, errlen, "paged_store: bad rows (T=%d, type=%d into a cache of type %d)", T, type, c->type);
        return -1;
    }
    if (!T) return 0;
    if (!k || !v || !slot) { snprintf(err, errlen, "paged_store: no rows or no slots"); return -1; }
    hipStream_t st;
    if (!stream_of(stream, st, "paged_store", err, errlen)) return -1;
    a.k = k; a.k_tok = k_tok; a.v = v; a.v_tok = v_tok;
    a.type = row_type(type); a.T = T; a.slot = slot;
    if (paged_store_launch(a, st)) { snprintf(err, errlen, "paged_store launch failed"); return -1; }
    return 0;
}

static bool batch_ok(int n_req, int T, int H, int Hkv, int window, int n_sink) {
    return n_req >= 0 && n_req <= kMaxReq && T >= 0 && Hkv >= 1 && Hkv <= 1024 && H >= Hkv && H % Hkv == 0 && (int64_t)T * H <= (1 << 27) &&
           (int64_t)std::min(n_req, T) * Hkv <= (1 << 22) &&   // a launch has fewer than 2^32 threads
           window >= 0 && n_sink >= 0;
}
static bool paged_batch_ok(const xjh_paged *c, int type, int T, int H, int n_req, int max_blocks) {
    return (type == XJ_F32 || type == c->type) && batch_ok(n_req, T, H, c->Hkv, 0, 0) && max_blocks >= 1 &&
           (int64_t)max_blocks * c->page <= (1 << 30);
}
static bool packed_batch_ok(int type, int T, int H, int Hkv, int D, int n_seq) {
    return row_type(type) >= 0 && batch_ok(n_seq, T, H, Hkv, 0, 0) && (D == 64 || D == 128 || D == 256);
}
static void batch_args(BatchAttnArgs &a, int type, int n_req, int T, int H, int Hkv, int D, int window, int n_sink) {
    a.type = row_type(type);
    a.n_req = n_req; a.T = T; a.H = H; a.Hkv = Hkv; a.D = D; a.G = H / Hkv;
    a.inv_g = UINT32_MAX / (uint32_t)a.G;
    a.window = window < (1 << 30) ? window : 0;   // positions are below 2^30
    a.sinks = n_sink;
}

extern "C" int xjh_attn_paged(const xjh_paged *c, int type, const void *q, int64_t q_tok, int64_t q_head, const void *gate,
                              int64_t g_tok, int64_t g_head, const int32_t *table, int max_blocks, const int32_t *cu,
                              const int32_t *kv_len, int n_req, int T, int max_new, int H, int window, int n_sink, float scale,
                              void *out, int64_t o_tok, void *work, size_t work_bytes, void *stream, char *err, size_t errlen) {
    Paged p;
    if (!cache_ok(c, "attn_paged", p, err, errlen)) return -1;
    if (!paged_batch_ok(c, type, T, H, n_req, max_blocks) || window < 0 || n_sink < 0 || !std::isfinite(scale)) {
        snprintf(err, errlen, "attn_paged: bad shape (type=%d over %d, n_req=%d, T=%d, H=%d on %d kv heads, max_blocks=%d, window=%d, n_sink=%d, scale=%g)",
                 type, c->type, n_req, T, H, c->Hkv, max_blocks, window, n_sink, scale);
        return -1;
    }
    if (!T || !n_req) return 0;
    if (!q || !out || !table || !cu || !kv_len || ((uintptr_t)work & 15)) {
        snprintf(err, errlen, "attn_paged: a buffer is missing, or an unaligned work area");
        return -1;
    }
    hipStream_t st;
    if (!stream_of(stream, st, "attn_paged", err, errlen)) return -1;
    BatchAttnArgs a{};
    batch_args(a, type, n_req, T, H, p.Hkv, p.D, window, n_sink);
    a.q = q; a.q_tok = q_tok; a.q_head = q_head;
    a.gate = gate; a.g_tok = g_tok; a.g_head = g_head;
    a.out = out; a.o_tok = o_tok;
    a.k = p.k; a.v = p.v;
    a.kv_type = p.bf16 ? kRowBf16 : kRowF16;
    a.table = table; a.kv_len = kv_len; a.cu = cu;
    a.lg = p.lg; a.n_pages = p.n_pages; a.max_blocks = max_blocks;
    a.max_new = max_new; a.scale = scale;
    a.part = (float *)work;
    if (batch_attn_launch(a, work ? (int64_t)(work_bytes / sizeof(float)) : 0, st)) {
        snprintf(err, errlen, "attn_paged launch failed");
        return -1;
    }
    return 0;
}

extern "C" size_t xjh_attn_paged_work_bytes(const xjh_paged *c, int type, int T, int H, int n_req, int max_new, int max_blocks) {
    if (!shape_ok(c) || !paged_batch_ok(c, type, T, H, n_req, max_blocks)) return 0;
    BatchAttnArgs a{};
    batch_args(a, type, n_req, T, H, c->Hkv, c->D, 0, 0);
    a.table = (const int32_t *)c;   // pages
    a.lg = __builtin_ctz((unsigned)c->page); a.max_blocks = max_blocks; a.max_new = max_new;
    return (size_t)batch_attn_part_floats(a) * sizeof(float);
}

extern "C" int xjh_attn_packed(int type, const void *q, int64_t q_tok, int64_t q_head, const void *k, int64_t k_tok, int64_t k_head,
                               const void *v, int64_t v_tok, int64_t v_head, const void *gate, int64_t g_tok, int64_t g_head,
                               const int32_t *cu, int n_seq, int T, int H, int Hkv, int D, int window, int n_sink, float scale,
                               void *out, int64_t o_tok, void *work, size_t work_bytes, void *stream, char *err, size_t errlen) {
    if (!packed_batch_ok(type, T, H, Hkv, D, n_seq) || window < 0 || n_sink < 0 || !std::isfinite(scale)) {
        snprintf(err, errlen, "attn_packed: bad shape (type=%d, n_seq=%d, T=%d, H=%d on %d kv heads of %d (64|128|256), window=%d, n_sink=%d, scale=%g)",
                 type, n_seq, T, H, Hkv, D, window, n_sink, scale);
        return -1;
    }
    if (!T || !n_seq) return 0;
    if (!q || !k || !v || !out || !cu || ((uintptr_t)work & 15)) {
        snprintf(err, errlen, "attn_packed: a buffer is missing, or an unaligned work area");
        return -1;
    }
    hipStream_t st;
    if (!stream_of(stream, st, "attn_packed", err, errlen)) return -1;
    BatchAttnArgs a{};
    batch_args(a, type, n_seq, T, H, Hkv, D, window, n_sink);
    a.q = q; a.q_tok = q_tok; a.q_head = q_head;
    a.gate = gate; a.g_tok = g_tok; a.g_head = g_head;
    a.out = out; a.o_tok = o_tok;
    a.k = k; a.k_tok = k_tok; a.k_head = k_head;
    a.v = v; a.v_tok = v_tok; a.v_head = v_head;
    a.kv_type = a.type;
    a.cu = cu;
    a.scale = scale;
    a.part = (float *)work;
    if (batch_attn_launch(a, work ? (int64_t)(work_bytes / sizeof(float)) : 0, st)) {
        snprintf(err, errlen, "attn_packed launch failed");
        return -1;
    }
    return 0;
}

extern "C" size_t xjh_attn_packed_work_bytes(int type, int T, int H, int Hkv, int D, int n_seq) {
    if (!packed_batch_ok(type, T, H, Hkv, D, n_seq)) return 0;
    BatchAttnArgs a{};
    batch_args(a, type, n_seq, T, H, Hkv, D, 0, 0);
    return (size_t)batch_attn_part_floats(a) * sizeof(float);
}
