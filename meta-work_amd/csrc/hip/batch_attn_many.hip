// Attention over pages or packed rows for requests of many rows (gfx950): prompts and pieces of them. See batch_attn.h.
#include "batch_attn.h"
#include <algorithm>

namespace xjk {

__device__ const u32x4 kZeros[1] = {};

// Lane l: 16 bytes at p to LDS offset off + 16 l; off is uniform over the wavefront.
__device__ __forceinline__ void dma16(const void *p, uint32_t off) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(off) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// LDS is as every wavefront left it; loads in flight stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Where the keys come from: pages, rows that 16 bytes at a time can be copied from, any other rows.
enum { kPages = 0, kRows16 = 1, kRowsAny = 2 };

// A row's 16-byte chunks lie permuted in LDS, so that what an instruction reads falls on all banks: 16 rows' chunk c of the keys,
// 4 rows' chunks 4 c .. 4 c + 3 of the values.
template <int D>
__device__ __forceinline__ int key_swz(int row) { return D >= 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int val_swz(int row) { return D >= 128 ? (row & 3) << 2 : (row >> 1 & 1) << 2; }

// A tile of 128 rows, 32 a wavefront; tiles of BN keys and values pass through LDS, the next one on its way meanwhile.
// Lane l: row l & 31, half h = l >> 5.
template <int D, class E, int NP, int NK, int RT, int SRC>
__global__ __launch_bounds__(256, D <= 128 && NP == 1 ? 2 : 1) void attn_many_kernel(const BatchAttnArgs a) {
    typedef typename Row<RT>::t R;
    constexpr int BN = many_keys(D), NB = BN / 32, NS = D / 16, ND = D / 32, CH = D / 8;
    constexpr int PLANE = BN * D * 2, TENSOR = NK * PLANE, BUF = 2 * TENSOR;
    constexpr int COPIES = BN * CH / 256;   // of 16 bytes a lane and tensor
    extern __shared__ __align__(1024) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    Item it;
    if (!find_item<kManyRows, BN, false>(a, blockIdx.x, it)) return;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const int R0 = it.tile * kManyRows, n_rows = it.s.rows * a.G;
    const int row = R0 + 32 * w + (lane & 31), tok = min(row / a.G, it.s.rows - 1), p = it.s.pos0 + tok;
    const int pf = it.s.pos0 + R0 / a.G, pl = it.s.pos0 + min((R0 + kManyRows - 1) / a.G, it.s.rows - 1);
    const int wf = it.s.pos0 + min((R0 + 32 * w) / a.G, it.s.rows - 1), wl = it.s.pos0 + min((R0 + 32 * w + 31) / a.G, it.s.rows - 1);
    const bool rows_here = R0 + 32 * w < n_rows;
    const Range g = range_of<BN>(a, pf, pl);
    const int i0 = (int)((int64_t)g.n * it.piece / it.pieces), i1 = (int)((int64_t)g.n * (it.piece + 1) / it.pieces);
    const int32_t *tab = SRC == kPages ? a.table + (int64_t)it.s.r * a.max_blocks : nullptr;

    // ---- a tile's keys and values into LDS: chunk (row, x ^ swizzle) of plane 0 .. NK - 1
    auto any_sees = [&](int j) { return j <= pl && (!a.window || j > pf - a.window || j < a.sinks); };
    auto copy = [&](int i, int buf) {
        const int j0 = g.tile(i) * BN;
#pragma unroll
        for (int n = 0; n < COPIES; n++) {
            const int c0 = (n * 4 + w) * 64, r0 = c0 / CH;   // the wavefront's chunks, all in rows of one page
            const int c = c0 + lane, r = c / CH, x = c % CH, j = j0 + r;
            const int page = SRC == kPages ? page_at(a, tab, j0 + r0) : 0;
            const bool use = page >= 0 && any_sees(j);
            const void *kp, *vp;
            if (SRC == kPages) {
                const int64_t at = (((((int64_t)page * a.Hkv + it.head) << a.lg) + (j & ((1 << a.lg) - 1)))) * D;
                kp = (const E *)a.k + at + 8 * (x ^ key_swz<D>(r));
                vp = (const E *)a.v + at + 8 * (x ^ val_swz<D>(r));
            } else {
                kp = (const E *)a.k + (it.s.start + j) * a.k_tok + it.head * a.k_head + 8 * (x ^ key_swz<D>(r));
                vp = (const E *)a.v + (it.s.start + j) * a.v_tok + it.head * a.v_head + 8 * (x ^ val_swz<D>(r));
            }
            // what no row sees counts for nothing, whatever lies there
            dma16(use ? kp : kZeros, base + buf * BUF + 16 * c0);
            dma16(use ? vp : kZeros, base + buf * BUF + TENSOR + 16 * c0);
        }
    };
    auto through_registers = [&](int i) {
        const int j0 = g.tile(i) * BN;
#pragma unroll 2
        for (int n = 0; n < COPIES; n++) {
            const int c = n * 256 + tid, r = c / CH, x = c % CH, j = j0 + r;
            const bool use = any_sees(j);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int64_t at = t ? (it.s.start + j) * a.v_tok + it.head * a.v_head : (it.s.start + j) * a.k_tok + it.head * a.k_head;
                char *to = lds + t * TENSOR + 16 * (r * CH + (x ^ (t ? val_swz<D>(r) : key_swz<D>(r))));
                if constexpr (RT == kRowF32) {
                    float f[8] = {};
                    if (use) {
                        const f32x8_u y = *(const f32x8_u *)((const float *)(t ? a.v : a.k) + at + 8 * x);
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] = y[e];
                    }
                    V8<E> q[NK];
                    planes<E, NK>(f, q);
#pragma unroll
                    for (int k = 0; k < NK; k++) *(V8<E> *)(to + k * PLANE) = q[k];
                } else {
                    u32x4 y = u32x4{0, 0, 0, 0};
                    if (use) y = *(const u32x4_u *)((const uint16_t *)(t ? a.v : a.k) + at + 8 * x);
                    *(u32x4 *)to = y;
                }
            }
        }
    };
    if (SRC != kRowsAny && i0 < i1) copy(i0, 0);

    // ---- queries, with the scale's sign; float ones over f16 scaled to 2^14 .. 2^15 before they become planes
    V8<E> q[NS][NP];
    float c = fabsf(a.scale) * 1.44269504088896340736f;
    {
        const R *x = (const R *)a.q + (it.s.start + tok) * a.q_tok + (it.head * a.G + min(row, n_rows - 1) % a.G) * a.q_head + 8 * h;
        float up = a.scale < 0.f ? -1.f : 1.f;
        if constexpr (NP == 2) {
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf((float)x[16 * s + i]));
            top = max_x32(top);
            int e = 15;
            if (top > 0.f && top < INFINITY) (void)frexpf(top, &e);
            e = max(e, -100);
            up = ldexpf(up, 15 - e);
            c = ldexpf(c, e - 15);
        }
#pragma unroll
        for (int s = 0; s < NS; s++) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = (float)x[16 * s + i] * up;
            planes<E, NP>(f, q[s]);
        }
    }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;   // m: a whole number, so that every rescaling is exact

    for (int i = i0; i < i1; i++) {
        const int buf = SRC == kRowsAny ? 0 : (i - i0) & 1, j0 = g.tile(i) * BN;
        if constexpr (SRC == kRowsAny) {
            lds_barrier();
            through_registers(i);
            __syncthreads();
        } else {
            if (i + 1 < i1) {
                copy(i + 1, buf ^ 1);
                wait_vm<2 * COPIES>();
            } else {
                wait_vm<0>();
            }
            lds_barrier();
        }
        const char *kb = lds + buf * BUF, *vb = kb + TENSOR;
        if (rows_here && j0 <= wl) {
            f32x16 s[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[b][r] = 0.f;
                const int kr = 32 * b + (lane & 31);
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    const char *at = kb + 16 * (kr * CH + ((2 * st + h) ^ key_swz<D>(kr)));
#pragma unroll
                    for (int k = NK - 1; k >= 0; k--) {
                        const V8<E> kf = *(const V8<E> *)(at + k * PLANE);
#pragma unroll
                        for (int n = (NK == 1 ? NP : NP - k) - 1; n >= 0; n--) s[b] = Op<E>::mfma32(kf, q[st][n], s[b]);
                    }
                }
            }
            bool full = j0 + BN - 1 <= wf && (!a.window || j0 > wl - a.window || j0 + BN - 1 < a.sinks);
            uint32_t page_ok = 0xFFFFFFFFu;   // a bit for 16 keys
            if (SRC == kPages) {
#pragma unroll
                for (int u = 0; u < BN / 16; u++)
                    if (page_at(a, tab, j0 + 16 * u) < 0) page_ok &= ~(1u << u);
                full = full && page_ok == 0xFFFFFFFFu;
            }
            uint32_t vis[NB];
            bool seen = true, bad = false;
            float top = -INFINITY;
            if (!full) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    vis[b] = 0;
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int kj = 32 * b + 8 * (r >> 2) + 4 * h + (r & 3);
                        if (sees(a, p, j0 + kj) && (page_ok >> (kj >> 4) & 1)) {
                            vis[b] |= 1u << r;
                            top = fmaxf(top, s[b][r]);
                        }
                    }
                }
                uint32_t any = 0;
#pragma unroll
                for (int b = 0; b < NB; b++) any |= vis[b];
                const unsigned long long all = __ballot(any != 0);
                seen = ((all >> (lane & 31) | all >> (32 + (lane & 31))) & 1) != 0;
                // values that are not finite make the rows that see them so, and no other (0 times infinity)
                for (int n = lane; n < TENSOR / 16; n += 64) {
                    const u32x4 y = *(const u32x4 *)(vb + 16 * n);
#pragma unroll
                    for (int k = 0; k < 4; k++) bad |= (y[k] & Op<E>::kExp) == Op<E>::kExp || (y[k] >> 16 & Op<E>::kExp) == Op<E>::kExp;
                }
                bad = __any(bad);
            } else {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int r = 0; r < 16; r++) top = fmaxf(top, s[b][r]);
            }
            top = max_x32(top);
            const float mn = fmaxf(m, seen ? fmaxf(ceilf(top * c), kLowest) : -INFINITY);
            if (__any(mn > m)) {
                const float up = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                l *= up;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= up;
                m = mn;
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    float pr[8];
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        pr[n] = __builtin_amdgcn_exp2f(fmaf(s[b][8 * t + n], c, Op<E>::kLift - m));
                        if (!full && !(vis[b] >> (8 * t + n) & 1)) pr[n] = 0.f;
                        l += pr[n];
                    }
                    V8<E> pp[NP];
                    planes<E, NP>(pr, pp);
                    // keys 32 b + 16 t + 4 h + (0 .. 3, 8 .. 11): this lane fetches 4 of one of them for the others
                    const int key = 32 * b + 16 * t + 4 * h + ((lane & 15) >> 2);
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const int chunk = 4 * d + 2 * (lane >> 4 & 1) + ((lane & 3) >> 1);
                        const char *at = vb + 16 * (key * CH + (chunk ^ val_swz<D>(key))) + 8 * (lane & 1);
                        const char *at8 = vb + 16 * ((key + 8) * CH + (chunk ^ val_swz<D>(key + 8))) + 8 * (lane & 1);
#pragma unroll
                        for (int k = NK - 1; k >= 0; k--) {
                            typedef short s16x4 __attribute__((ext_vector_type(4)));
                            typedef __attribute__((address_space(3))) s16x4 *lp;
                            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at + k * PLANE)));
                            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at8 + k * PLANE)));
                            u32x4 v = u32x4{x[0], x[1], y[0], y[1]};
                            if (bad) {
                                u32x4 mark, sight;
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const bool lo = (v[e] & Op<E>::kExp) == Op<E>::kExp, hi = (v[e] >> 16 & Op<E>::kExp) == Op<E>::kExp;
                                    mark[e] = (lo ? Op<E>::kOne : 0u) | (hi ? Op<E>::kOne << 16 : 0u);
                                    v[e] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
                                    const uint32_t bits = full ? 3u : vis[b] >> (8 * t + 2 * e);
                                    sight[e] = (bits & 1 ? Op<E>::kOne : 0u) | (bits & 2 ? Op<E>::kOne << 16 : 0u);
                                }
                                f32x16 z;
#pragma unroll
                                for (int r = 0; r < 16; r++) z[r] = 0.f;
                                z = Op<E>::mfma32(__builtin_bit_cast(V8<E>, mark), __builtin_bit_cast(V8<E>, sight), z);
#pragma unroll
                                for (int r = 0; r < 16; r++) o[d][r] += z[r] > 0.f ? NAN : 0.f;
                            }
#pragma unroll
                            for (int n = (NK == 1 ? NP : NP - k) - 1; n >= 0; n--)
                                o[d] = Op<E>::mfma32(__builtin_bit_cast(V8<E>, v), pp[n], o[d]);
                        }
                    }
                }
        }
        if (SRC != kRowsAny) lds_barrier();
    }
    l += __shfl_xor(l, 32, 64);
    if (row >= n_rows) return;
    if (it.pieces > 1) {
        const int64_t at = (int64_t)it.slot * kManyRows + row - R0;
        if (h == 0) *part_stat(a, at, kManyRows, D) = float2{m, l};
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(f32x4 *)(part_sums(a, at, D) + 32 * d + 8 * r + 4 * h) = f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
        return;
    }
    const int head = it.head * a.G + row % a.G;
    R *out = (R *)a.out + (it.s.start + tok) * a.o_tok + head * D + 4 * h;
    const R *gate = a.gate ? (const R *)a.gate + (it.s.start + tok) * a.g_tok + head * a.g_head + 4 * h : nullptr;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            float z = m == -INFINITY ? 0.f : o[d][r] / l;
            const int at = 32 * d + 8 * (r >> 2) + (r & 3);
            if (gate) z *= xjd::sigm((float)gate[at]);
            out[at] = (R)z;
        }
}

template <int D, class E, int NP, int NK, int RT, int SRC>
static int many(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    constexpr int bytes = 2 * NK * many_keys(D) * D * 2 * (SRC == kRowsAny ? 1 : 2);
    auto *f = attn_many_kernel<D, E, NP, NK, RT, SRC>;
    if (bytes > 65536 && hipFuncSetAttribute((const void *)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return -1;
    f<<<dim3((unsigned)items), 256, bytes, st>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int D>
static int many(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    if (a.table) {
        if (a.type == kRowF16) return many<D, _Float16, 1, 1, kRowF16, kPages>(a, items, st);
        if (a.type == kRowBf16) return many<D, __bf16, 1, 1, kRowBf16, kPages>(a, items, st);
        if (a.kv_type == kRowF16) return many<D, _Float16, 2, 1, kRowF32, kPages>(a, items, st);
        return many<D, __bf16, 3, 1, kRowF32, kPages>(a, items, st);
    }
    if (a.type == kRowF32) return many<D, __bf16, 3, 3, kRowF32, kRowsAny>(a, items, st);
    const bool whole = !(((uintptr_t)a.k | (uintptr_t)a.v) & 15) && !((a.k_tok | a.k_head | a.v_tok | a.v_head) & 7);
    if (a.type == kRowF16) {
        return whole ? many<D, _Float16, 1, 1, kRowF16, kRows16>(a, items, st) : many<D, _Float16, 1, 1, kRowF16, kRowsAny>(a, items, st);
    }
    return whole ? many<D, __bf16, 1, 1, kRowBf16, kRows16>(a, items, st) : many<D, __bf16, 1, 1, kRowBf16, kRowsAny>(a, items, st);
}
int attn_many_launch(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    return a.D == 64 ? many<64>(a, items, st) : a.D == 128 ? many<128>(a, items, st) : many<256>(a, items, st);
}

// ---------------------------------------------------------------- launch --

// Few rows: the kernel that reads keys straight into registers takes requests whose new tokens fill at most two of its tiles.
static bool few_rows(const BatchAttnArgs &a) {
    return a.table && a.max_new > 0 && (int64_t)a.max_new * a.G <= 2 * kFewRows;
}
// Row tiles times heads, at most.
static int64_t tiles_bound(const BatchAttnArgs &a, int BM) {
    return ((int64_t)a.T * a.G / BM + std::min(a.n_req, a.T)) * a.Hkv;
}
struct Split {
    int BM, target, least;
    int64_t tiles, items;
};
// Pieces aimed at: enough for every CU.
static Split split_of(const BatchAttnArgs &a) {
    Split s;
    const bool few = few_rows(a);
    s.BM = few ? kFewRows : kManyRows;
    s.tiles = tiles_bound(a, s.BM);
    const int BN = few ? kFewKeys : many_keys(a.D);
    s.least = few ? 8 : 8;
    const int64_t longest = ((a.table ? (int64_t)a.max_blocks << a.lg : a.T) + BN - 1) / BN;
    s.target = longest <= s.least || s.tiles > 1024 ? 0 : 512;
    s.items = s.target ? std::min(s.tiles * ((longest + s.least - 1) / s.least), s.tiles + s.target) : s.tiles;
    return s;
}
static int64_t slot_floats(const BatchAttnArgs &a, int BM) { return (int64_t)BM * (a.D + 2); }

int64_t batch_attn_part_floats(const BatchAttnArgs &a) {
    const Split s = split_of(a);
    return s.target ? std::min<int64_t>(s.items, 2 * s.target) * slot_floats(a, s.BM) : 0;
}

int batch_attn_launch(const BatchAttnArgs &args, int64_t part_floats, hipStream_t st) {
    BatchAttnArgs a = args;
    Split s = split_of(a);
    a.slots = (int)std::min<int64_t>(part_floats / slot_floats(a, s.BM), 1 << 20);
    a.target = std::min(s.target, a.slots / 2);   // at most 2 a.target items in pieces
    a.least = s.least;
    const int64_t items = a.target ? std::min(s.items, s.tiles + a.target) : s.tiles;
    if (s.BM == kFewRows ? attn_few_launch(a, items, st) : attn_many_launch(a, items, st)) return -1;
    return a.target ? attn_merge_launch(a, s.BM, std::min<int64_t>(s.tiles, a.target), st) : 0;
}

}  // namespace xjk
