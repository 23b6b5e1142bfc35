// A key/value cache in pages (gfx950): who owns which page (xjh_page_plan), and new rows into their slots (xjh_paged_store).
#include "common.h"
#include "kernels.h"
#include <algorithm>

namespace xjk {

// ------------------------------------------------------------- page plan --

// A request's row of the table: `have` blocks are there, `need` will be, `past` tokens before `fresh` new ones.
struct Req {
    int past, fresh, have, need, kv;
    int64_t beyond;   // positions that do not fit the row
};
__device__ __forceinline__ Req request(const PlanArgs &a, int r) {
    const int L = a.max_blocks << a.lg, up = (1 << a.lg) - 1;
    Req q;
    q.past = min(max(a.n_past[r], 0), L);
    q.fresh = max(a.n_new[r], 0);
    const int held = a.held ? min(max(a.held[r], 0), L) : q.past;
    const int64_t n = (int64_t)q.past + q.fresh;
    q.kv = (int)min(n, (int64_t)L);
    q.beyond = n - q.kv;
    q.have = (int)(((int64_t)held + up) >> a.lg);
    q.need = (int)(((int64_t)q.kv + up) >> a.lg);
    return q;
}
// The last of n entries cu[0] = 0 <= cu[1] <= .. with cu[i] <= x (x >= 0), that is the one whose run holds x.
__device__ __forceinline__ int run_of(const int32_t *cu, int n, int x) {
    int lo = 0, hi = n;   // cu[lo] <= x < cu[hi]
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (cu[m] <= x) lo = m;
        else hi = m;
    }
    return lo;
}

constexpr int kPlanThreads = 1024;

// Sums over the requests before each: rows, pages given back, pages taken. One work-group, the requests in runs of its threads. (Rows in
// two halves of 16 bits: their sum may pass 32.)
__device__ __forceinline__ void plan_scan(const PlanArgs &a) {
    constexpr int W = kPlanThreads / 64;
    __shared__ int red[4][W];
    __shared__ int64_t over[W];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int64_t rows = 0, beyond = 0;
    int base[2] = {0, 0};
    for (int r0 = 0; r0 < a.n_req; r0 += kPlanThreads) {
        const int r = r0 + tid;
        Req q{};
        if (r < a.n_req) q = request(a, r);
        beyond += q.beyond;
        int x[4] = {q.fresh & 0xFFFF, q.fresh >> 16, max(q.have - q.need, 0), max(q.need - q.have, 0)}, all[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = xjd::wave_scan(x[i]);
            if (lane == 63) red[i][w] = x[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int own = red[i][lane % W], to = xjd::row16_scan(own);
            x[i] += __builtin_amdgcn_readlane(to - own, w);
            all[i] = __builtin_amdgcn_readlane(to, W - 1);
        }
        if (r < a.n_req) {
            a.cu[r + 1] = (int)min(rows + x[0] + ((int64_t)x[1] << 16), (int64_t)INT32_MAX);
            a.rel_cu[r + 1] = base[0] + x[2];
            a.take_cu[r + 1] = base[1] + x[3];
            a.kv_len[r] = q.kv;
        }
        rows += all[0] + ((int64_t)all[1] << 16);
        base[0] += all[2];
        base[1] += all[3];
        __syncthreads();
    }
    if (__any(beyond != 0))
        for (int o = 32; o; o >>= 1) beyond += __shfl_xor(beyond, o, 64);
    if (lane == 0) over[w] = beyond;
    __syncthreads();
    if (tid == 0) {
        beyond = 0;
        for (int k = 0; k < W; k++) beyond += over[k];
        const int n_free = min(max(*a.n_free, 0), a.n_pages);
        const int all = (int)min((int64_t)n_free + base[0], (int64_t)a.n_pages), takes = base[1];
        const int left = takes > all ? all : all - takes;   // pages missing: none is taken
        const int64_t big = INT32_MAX;
        a.cu[0] = a.rel_cu[0] = a.take_cu[0] = 0;
        a.sum[0] = n_free;
        a.sum[1] = all;
        a.sum[2] = left;
        a.sum[3] = takes;
        *a.n_free_out = left;
        a.status[0] = max(takes - all, 0);
        a.status[1] = (int)min(beyond, big);
        a.status[2] = (int)min(max(rows - a.T, (int64_t)0), big);
        a.status[3] = (int)min(rows, big);
    }
}
// Entry i of the free pages with those given back behind them.
__device__ __forceinline__ int stack_at(const PlanArgs &a, int n_free, int i) {
    if (i < n_free) return a.free_list[i];
    const int k = i - n_free, r = run_of(a.rel_cu, a.n_req, k);
    return a.table[(int64_t)r * a.max_blocks + request(a, r).need + k - a.rel_cu[r]];
}
// The pages that move (what 1: taken, 2: given back), and the rows' positions and slots (4), each by a thread of its own. What is read here of the
// table and of the free list is not what is written: rows give or take, and pages are taken from `left` on, put back below it. cu: the requests'
// first rows, the array or a copy in LDS.
__device__ __forceinline__ void plan_expand(const PlanArgs &a, int what, const int32_t *cu) {
    const int n_free = a.sum[0], all = a.sum[1], left = a.sum[2], takes = a.sum[3];
    const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    auto taken = [&](int i) { return takes <= all ? stack_at(a, n_free, all - 1 - i) : -1; };
    if (what & 1)
        for (int64_t i = first; i < takes; i += step) {
            const int r = run_of(a.take_cu, a.n_req, (int)i);
            a.table[(int64_t)r * a.max_blocks + request(a, r).have + (int)i - a.take_cu[r]] = taken((int)i);
        }
    if (what & 2)
        for (int64_t i = n_free + first; i < left; i += step) a.free_list[i] = stack_at(a, n_free, (int)i);
    if (what & 4) {
        const int rows = a.n_req ? cu[a.n_req] : 0;
        for (int64_t t = first; t < a.T; t += step) {
            int pos = 0, slot = -1;
            if (t < rows) {
                const int r = run_of(cu, a.n_req, (int)t);
                const Req q = request(a, r);
                const int64_t p = (int64_t)q.past + (t - cu[r]);
                pos = (int)min(p, (int64_t)INT32_MAX);
                if (p < q.kv) {
                    const int b = (int)(p >> a.lg);
                    const int page = b < q.have ? a.table[(int64_t)r * a.max_blocks + b] : taken(a.take_cu[r] + b - q.have);
                    if (page >= 0 && page < a.n_pages) slot = (page << a.lg) + (int)(p & ((1 << a.lg) - 1));
                }
            }
            if (a.pos) a.pos[t] = pos;
            if (a.slot) a.slot[t] = slot;
        }
    }
}
__global__ __launch_bounds__(kPlanThreads) void plan_scan_kernel(const PlanArgs a) { plan_scan(a); }
// Work-groups of one kind each, so that no thread waits for one chain of loads after the other (1000 requests with 153600 rows 11 -> 8 us, the
// requests' first rows searched in LDS).
constexpr int kPlanLds = 4096;
__global__ __launch_bounds__(256) void plan_expand_kernel(const PlanArgs a) {
    __shared__ int32_t cu[kPlanLds + 1];
    const int what = 1 << blockIdx.y;
    if (what == 4 && a.n_req <= kPlanLds) {
        for (int i = threadIdx.x; i <= a.n_req; i += 256) cu[i] = a.cu[i];
        __syncthreads();
        plan_expand(a, what, cu);
    } else {
        plan_expand(a, what, a.cu);
    }
}
// All of it in one work-group: what it wrote it reads back behind a barrier.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const PlanArgs a) {
    plan_scan(a);
    __threadfence_block();
    __syncthreads();
    plan_expand(a, 7, a.cu);
}

int page_plan_launch(const PlanArgs &a, hipStream_t st) {
    // A second launch costs what a thread's four rows do (8 requests of a token each 5.2 + 2.9 us in two, 4.2 in one). The pages that move are not known here:
    // those taken are few where the rows are, but requests that end give back all of theirs, a thread some 0.7 us each (8 of 131000 positions in pages
    // of 16: 52 us a call, 10.5 in two launches; 64 of 4000 20 and 10.5). So one launch only where there are no more pages than cost some 50 us.
    const int64_t pages = std::min<int64_t>(a.n_pages, (int64_t)a.n_req * a.max_blocks);
    if (a.n_req <= 256 && a.T <= 4 * kPlanThreads && pages <= 64 * kPlanThreads) {
        plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
    } else {
        plan_scan_kernel<<<1, kPlanThreads, 0, st>>>(a);
        plan_expand_kernel<<<dim3(std::min(1024, std::max(64, (a.T + 255) / 256)), 3), 256, 0, st>>>(a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ----------------------------------------------------------------- store --

typedef unsigned short us8 __attribute__((ext_vector_type(8)));
typedef unsigned short us8_u __attribute__((ext_vector_type(8), aligned(2)));   // rows of any 2-byte alignment
typedef float f32x8_u __attribute__((ext_vector_type(8), aligned(4)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// A thread moves 8 elements of a row. Bound by memory (8000 rows of 8 heads of 128 in bf16, 33 MB in and 33 out, 11.1 us, 5.9 TB/s: the pages
// stay in the memory-side cache) or the launch (16 float rows of 4 heads of 256 2.3 us).
template <int TYPE, bool BF>
__global__ __launch_bounds__(256) void paged_store_kernel(const PagedStoreArgs a) {
    const int per = a.c.Hkv * a.c.D / 8;   // pieces of a row
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.T * per) return;
    const int t = (int)(i / per), c = (int)(i - (int64_t)t * per) * 8, slot = a.slot[t];
    if (slot < 0 || (slot >> a.c.lg) >= a.c.n_pages) return;
    const void *x = blockIdx.y ? a.v : a.k;
    const int64_t at = t * (blockIdx.y ? a.v_tok : a.k_tok) + c;
    us8 y;
    if constexpr (TYPE == kRowF32) {
        const f32x8_u f = *(const f32x8_u *)((const float *)x + at);
        if constexpr (BF) y = __builtin_bit_cast(us8, __builtin_convertvector(f, bf8));
        else y = __builtin_bit_cast(us8, __builtin_convertvector(f, hf8));
    } else {
        y = *(const us8_u *)((const unsigned short *)x + at);
    }
    const int h = c / a.c.D, d = c - h * a.c.D;
    unsigned short *out = (unsigned short *)(blockIdx.y ? a.c.v : a.c.k);
    const int64_t row = ((((int64_t)(slot >> a.c.lg) * a.c.Hkv + h) << a.c.lg) + (slot & ((1 << a.c.lg) - 1)));
    *(us8 *)(out + row * a.c.D + d) = y;
}

int paged_store_launch(const PagedStoreArgs &a, hipStream_t st) {
    const int64_t n = (int64_t)a.T * (a.c.Hkv * a.c.D / 8);
    const dim3 grid((unsigned)((n + 255) / 256), 2);
    if (a.type == kRowF32 && a.c.bf16) paged_store_kernel<kRowF32, true><<<grid, 256, 0, st>>>(a);
    else if (a.type == kRowF32) paged_store_kernel<kRowF32, false><<<grid, 256, 0, st>>>(a);
    else paged_store_kernel<kRowF16, false><<<grid, 256, 0, st>>>(a);   // 16 bits of either type as they are
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace xjk
