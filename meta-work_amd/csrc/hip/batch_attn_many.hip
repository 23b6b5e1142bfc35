// Attention over pages or packed rows for requests of many rows (gfx950): prompts and pieces of them. See batch_attn.h.
#include "batch_attn.h"
#include <algorithm>
#include <type_traits>

namespace xjk {

__device__ const u32x4 kZeros[2] = {};

// Lane l: 16 bytes at p to LDS offset off + 16 l; off is uniform over the wavefront.
__device__ __forceinline__ void dma16(const void *p, uint32_t off) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(off) : "memory", "m0");
}
// The same with a uniform base and a lane's offset from it.
__device__ __forceinline__ void dma16(const void *base, uint32_t lane_off, uint32_t off) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_off), "s"(base), "s"(off) : "memory", "m0");
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

// Where the keys come from: pages, or rows that can be copied 16 bytes at a time.
enum { kPages = 0, kRows16 = 1 };

template <class T>
__device__ __forceinline__ T lds_read(uint32_t at, uint32_t off) {
    return *(const __attribute__((address_space(3))) T *)(uintptr_t)(at + off);
}
// Of 16 lanes, each at 4 dims of a key (l / 4 % 4 of 4 keys): the four keys of dim l % 16.
__device__ __forceinline__ u32x2 lds_read_turned(uint32_t at, uint32_t off) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)(at + off)));
}
// The lane's number, anew: what is made of it is not kept in registers from one use to the next.
__device__ __forceinline__ int fresh_lane() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
}
// What a wavefront holds of its M rows, 32 or 16, on the instruction of M by M by 512 / M. Lane l: row l % M, part h = l / M of the keys.
// With 32 rows every operand read from LDS feeds one instruction of 32 clocks, which is as fast as LDS can be; it needs D / 2 registers for the sums and
// D / 4 for the queries, with 256 dims just within the 256 that two wavefronts a SIMD leave it (a register that lies in memory instead is waited for
// behind the tiles on their way). With 16 rows it is half of each: for float rows, whose planes use an operand two or three times.
template <int D, class E, int NP, int NK, class R, int M>
struct WaveRows {
    static constexpr int BN = many_keys(D), NS = D * M / 512, ND = D / M, CH = D / 8, KI = 512 / M;   // KI: keys a step of the second product
    static constexpr int PER = M * M / 64, NB = BN / M, NE = NB * PER;                                  // scores a block, blocks, scores a lane
    static constexpr int PLANE = BN * D * 2, TENSOR = NK * PLANE;
    static constexpr int QL = D < 256 ? 0 : M == 32 ? 3 : NK == 3 ? 7 : 0;   // steps whose queries' last plane lies in LDS, as far as that is free
    typedef float F __attribute__((ext_vector_type(PER)));
    V8<E> q[NS][NP];
    uint32_t q_lds;   // where the wavefront's first QL steps lie
    F o[ND];
    float m, l, c;   // the reference in powers of two (a whole number, so that every rescaling is exact), the weights' sum, the scale
    float lift;      // with NP = 3 as a factor behind the exponential: a far exponent would round its argument
    int lane, h;

    static __device__ __forceinline__ F mfma(V8<E> a, V8<E> b, F x) {
        if constexpr (M == 32) return Op<E>::mfma32(a, b, x);
        else return Op<E>::mfma16(a, b, x);
    }
    static __device__ __forceinline__ int key_of(int e, int h) {   // of a lane's element e
        const int r = e % PER;
        return M * (e / PER) + 8 * (r >> 2) + 4 * h + (r & 3);
    }
    static __device__ __forceinline__ float most(float x) { return M == 32 ? max_x32(x) : max_x32(max_x16(x)); }
    // A row's 16-byte chunks lie permuted in LDS, so that what an instruction reads falls on all banks: 16 rows' chunk c of the keys;
    // of the values 4 rows' chunks 4 c .. 4 c + 3 (M = 32), 8 rows' chunks 2 c, 2 c + 1 (M = 16).
    static __device__ __forceinline__ int key_swz(int row) { return D >= 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int val_swz(int row) {
        if (D < 128) row >>= 1;
        return M == 32 ? (row & (D >= 128 ? 3 : 1)) << 2 : (row & (D >= 128 ? 7 : 3)) << 1;
    }

    // Queries, with the scale's sign; float ones over f16 scaled to 2^14 .. 2^15 before they become planes.
    __device__ __forceinline__ void start(const R *qp, float scale, uint32_t q_area, const Seq &seq) {
        lane = threadIdx.x & 63;
        h = lane / M;
        q_lds = q_area + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024 * QL;
        c = fabsf(scale) * 1.44269504088896340736f;
        float up = scale < 0.f ? -1.f : 1.f;
        Rows<R, 8> x[NS];
#pragma unroll
        for (int s = 0; s < NS; s++) x[s] = *(const Rows<R, 8> *)(qp + KI * s + 8 * h);
        if constexpr (NP == 2) {
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf((float)x[s][i]));
            top = most(top);
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
            for (int i = 0; i < 8; i++) f[i] = (float)x[s][i] * up;
            planes<E, NP>(f, q[s]);
            if (s < QL) *(__attribute__((address_space(3))) V8<E> *)(uintptr_t)(q_lds + 1024 * s + 16 * lane) = q[s][NP - 1];
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < PER; r++) o[d][r] = 0.f;
        m = -INFINITY;
        l = 0.f;
        lift = lift_of<E, BN>(seq);
        if (NP == 3) lift = __builtin_amdgcn_exp2f(lift);
    }
    // Scores of a tile whose keys begin at LDS address kb.
    __device__ __forceinline__ void scores(uint32_t kb, F (&s)[NB]) const {
        const int lane = QL ? fresh_lane() : this->lane, kr = lane % M, h = lane / M;
        const uint32_t at = (kb + kr * 2 * D) | (16 * (h ^ key_swz(kr)));   // chunk KI / 8 * st + h: exclusive or with 2 KI st
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int r = 0; r < PER; r++) s[b][r] = 0.f;
#pragma unroll
            for (int st = 0; st < NS; st++)
#pragma unroll
                for (int k = NK - 1; k >= 0; k--) {
                    const V8<E> kf = lds_read<V8<E>>(at ^ (2 * KI * st), k * PLANE + 2 * M * b * D);
#pragma unroll
                    for (int n = (NK == 1 ? NP : NP - k) - 1; n >= 0; n--)
                        s[b] = mfma(kf, st < QL && n == NP - 1 ? lds_read<V8<E>>(q_lds + 16 * lane, 1024 * st) : q[st][n], s[b]);
                }
        }
    }
    // The running maximum with this tile's scores. (One that underflows every weight counts as seen.)
    template <bool MASKED>
    __device__ __forceinline__ void raise(const F (&s)[NB], uint32_t vis, bool seen) {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < NE; e++)
            if (!MASKED || (vis >> e & 1)) top = fmaxf(top, s[e / PER][e % PER]);
        top = most(top);
        const float now = !MASKED || seen ? fmaxf(ceilf(top * c), kLowest) : -INFINITY;
        const bool higher = now > m + Op<E>::kTol;
        if (__builtin_expect(__any(higher), 0)) {
            const float mn = higher ? now : m, up = higher ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
            l *= up;
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= up;
            m = mn;
        }
    }
    // Weights and sums. Those of 16-bit rows (NP = 1) are rounded to the type here, in their sum l they are not: with a second plane 8200 rows of 32 heads
    // on 8 of 128 in bf16 take 744 us for 571 and are off by 1.66e-3, which is the result's rounding, for 1.82e-3 (a piece of 512 rows at 32000 511 for 442,
    // 1.66e-3 for 1.72e-3).
    template <bool MASKED>
    __device__ __forceinline__ void weigh(uint32_t vb, const F (&s)[NB], uint32_t vis) {
        const float zero = NP == 3 ? -m : lift - m;
        // the lane fetches 4 dims of one key of a step's first (second) half for the others
        const int lane = QL ? fresh_lane() : this->lane, h = lane / M, key = 4 * h + (lane >> 2 & 3), low = (M == 32 ? 32 * (lane >> 4 & 1) : 0) + 8 * (lane & 3);
        const uint32_t at = (vb + key * 2 * D) | (low ^ 16 * val_swz(key));
        constexpr int DX = 128 / M;   // dims within which chunks are permuted, over M
#pragma unroll
        for (int u = 0; u < NE / 8; u++) {
            float pr[8];
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const int e = 8 * u + n;
                pr[n] = __builtin_amdgcn_exp2f(fmaf(s[e / PER][e % PER], c, zero));
                if (NP == 3) pr[n] *= lift;
                if (MASKED && !(vis >> e & 1)) pr[n] = 0.f;
                l += pr[n];
            }
            V8<E> pp[NP];
            planes<E, NP>(pr, pp);
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int k = NK - 1; k >= 0; k--) {
                    const uint32_t from = at ^ (2 * M * (d % DX)), off = k * PLANE + 256 * (d / DX) + KI * u * 2 * D;
                    const u32x2 x = lds_read_turned(from, off), y = lds_read_turned(from, off + 256 / M * 2 * D);
                    const V8<E> v = __builtin_bit_cast(V8<E>, u32x4{x[0], x[1], y[0], y[1]});
#pragma unroll
                    for (int n = (NK == 1 ? NP : NP - k) - 1; n >= 0; n--) o[d] = mfma(v, pp[n], o[d]);
                }
        }
    }
    // Which keys of a tile this lane's row sees, a bit an element; page_ok: a bit for 16 keys. Whether the row sees any.
    __device__ __forceinline__ bool look(const BatchAttnArgs &a, int p, int j0, uint32_t page_ok, uint32_t &vis) const {
        vis = 0;
#pragma unroll
        for (int e = 0; e < NE; e++) {
            const int kj = key_of(e, h);
            if (sees(a, p, j0 + kj) && (page_ok >> (kj >> 4) & 1)) vis |= 1u << e;
        }
        unsigned long long all = __ballot(vis != 0);
        all |= all >> 32;
        if (M == 16) all |= all >> 16;
        return (all >> (lane % M) & 1) != 0;
    }
    // Values that are not finite make the rows that see them so, and no other, where 0 times infinity would not do: the work-group
    // takes them out of a tile that some row does not see whole and leaves marks [BN][CH], a bit for each of a chunk's 8 dims, from which the
    // rows take them.
    __device__ __forceinline__ static bool find_spoilt(const char *vb) {
        uint32_t bad = 0;
        for (int n = threadIdx.x; n < TENSOR / 16; n += blockDim.x) {
            const u32x4 y = *(const u32x4 *)(vb + 16 * n);
#pragma unroll
            for (int k = 0; k < 4; k++) bad |= ((y[k] & Op<E>::kExp) == Op<E>::kExp) | ((y[k] >> 16 & Op<E>::kExp) == Op<E>::kExp);
        }
        return bad != 0;
    }
    __device__ static __attribute__((noinline)) void mark_spoilt(char *vb, uint8_t *marks) {
        for (int n = threadIdx.x; n < BN * CH; n += blockDim.x) {
            const int key = n / CH, x = n % CH;
            uint32_t mark = 0;
            for (int k = 0; k < NK; k++) {
                u32x4 *at = (u32x4 *)(vb + k * PLANE + 16 * (key * CH + (x ^ val_swz(key))));
                u32x4 y = *at;
                for (int e = 0; e < 4; e++) {
                    const bool lo = (y[e] & Op<E>::kExp) == Op<E>::kExp, hi = (y[e] >> 16 & Op<E>::kExp) == Op<E>::kExp;
                    mark |= (uint32_t)lo << (2 * e) | (uint32_t)hi << (2 * e + 1);
                    y[e] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
                }
                *at = y;
            }
            marks[n] = (uint8_t)mark;
        }
    }
    __device__ __forceinline__ void take_spoilt(const BatchAttnArgs &a, int p, int j0, uint32_t page_ok, const uint8_t *marks) {
#pragma unroll 1
        for (int key = 0; key < BN; key++) {
            const bool see = sees(a, p, j0 + key) && (page_ok >> (key >> 4) & 1);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                uint32_t w;
                if constexpr (M == 32) w = *(const uint32_t *)(marks + key * CH + 4 * d);
                else w = *(const uint16_t *)(marks + key * CH + 2 * d);
                w = see ? w >> (4 * h) : 0u;
                if (__any(w != 0))
#pragma unroll
                    for (int r = 0; r < PER; r++)
                        if (w >> (8 * (r >> 2) + (r & 3)) & 1) o[d][r] = NAN;
            }
        }
    }
    // The rows' results, or their part of them.
    __device__ __forceinline__ void finish(const BatchAttnArgs &a, const Item &it, int row, int tok) {
        if (M == 16) l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (row >= it.s.rows * a.G) return;
        if (it.pieces > 1) {
            const int64_t at = (int64_t)it.slot * kManyRows + row - it.tile * kManyRows;
            if (h == 0) *part_stat(a, at, kManyRows, D) = float2{m, l};
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int r = 0; r < PER / 4; r++)
                    *(f32x4 *)(part_sums(a, at, D) + M * d + 8 * r + 4 * h) = f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
            return;
        }
        const int head = it.head * a.G + row - tok * a.G;
        R *out = (R *)a.out + (it.s.start + tok) * a.o_tok + (int64_t)head * D + 4 * h;
        const R *gate = a.gate ? (const R *)a.gate + (it.s.start + tok) * a.g_tok + head * a.g_head + 4 * h : nullptr;
        const float inv = m == -INFINITY ? 0.f : 1.f / l;   // a row that has seen nothing is 0
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int r = 0; r < PER / 4; r++)
                finish4(f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]}, inv, gate ? gate + M * d + 8 * r : nullptr,
                        out + M * d + 8 * r);
    }
};
// LDS beside the tiles: marks of values that are not finite, and whether there are any.
constexpr int many_marks(int D) { return many_keys(D) * D / 8; }

// A tile of 128 rows, M a wavefront; tiles of BN keys and values pass through LDS. Each tile's sums are followed by the next one's scores, whose keys are
// there already, and the keys behind it and its values are on their way: a barrier a tile. Two work-groups a CU: while one's wavefront has the vector
// units for its softmax, the other's has the matrix cores. Bound by a wavefront's chain of operand reads, products and softmax: 8200 rows of 32 heads on 8
// of 128 in bf16 568 us (924 TFLOP/s), 512 rows behind 32000 of 16 on 4 of 256 369 with the join (733), calls back to back.
template <int D, class E, int NP, int RT, int SRC, int M>
__global__ __launch_bounds__(8192 / M, 2) void attn_many_kernel(const BatchAttnArgs a) {
    typedef typename Row<RT>::t R;
    typedef WaveRows<D, E, NP, 1, R, M> X;
    constexpr int BN = X::BN, NB = X::NB, CH = X::CH, TENSOR = X::TENSOR;
    constexpr int W = kManyRows / M, COPIES = BN * CH / (64 * W);   // wavefronts; copies of 16 bytes a lane and tensor
    extern __shared__ __align__(1024) char lds[];   // keys, keys, values, values, marks, flag
    uint8_t *const marks = (uint8_t *)lds + 4 * TENSOR;
    int *const flag = (int *)(marks + many_marks(D));
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    Item it;
    if (!find_item<kManyRows, BN, false>(a, blockIdx.x, it)) return;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const int R0 = it.tile * kManyRows, n_rows = it.s.rows * a.G;
    const int row = R0 + M * w + (X::QL ? fresh_lane() : lane) % M, rq = min(row, n_rows - 1), tok = token_of(a, rq);
    const int pf = it.s.pos0 + token_of(a, R0), pl = it.s.pos0 + token_of(a, min(R0 + kManyRows, n_rows) - 1);
    const int wl = it.s.pos0 + token_of(a, min(R0 + M * w + M, n_rows) - 1);
    const Range g = range_of<BN>(a, pf, pl);
    const int i0 = part_from(g.n, it.piece, it.pieces), n_tiles = part_from(g.n, it.piece + 1, it.pieces) - i0;
    const int32_t *tab = SRC == kPages ? a.table + (int64_t)it.s.r * a.max_blocks : nullptr;

    // ---- a tile's keys or values into LDS: chunk (row, x ^ swizzle). A wavefront's copy is of 64 chunks, in rows r0 .. of one page;
    // its lanes' offsets are of two kinds at most (the keys' with D = 256: odd copies)
    const uint32_t k_row = 2 * (SRC == kPages ? D : (uint32_t)a.k_tok), v_row = 2 * (SRC == kPages ? D : (uint32_t)a.v_tok);   // bytes
    const int64_t first = SRC == kPages ? ((int64_t)it.head << a.lg) * D : 0;
    const char *const k_base = (const char *)((const E *)a.k + (SRC == kPages ? first : it.s.start * a.k_tok + it.head * a.k_head));
    const char *const v_base = (const char *)((const E *)a.v + (SRC == kPages ? first : it.s.start * a.v_tok + it.head * a.v_head));
    const int64_t page_bytes = ((int64_t)a.Hkv << a.lg) * (2 * D);
    const int page_mask = (1 << a.lg) - 1;
    auto whole_tile = [&](int f, int l, int j0) __attribute__((always_inline)) { return j0 + BN - 1 <= f && (!a.window || j0 > l - a.window || j0 + BN - 1 < a.sinks); };
    // the pages of a tile, one for 16 positions (no array: indexed, it would lie in memory), asked for three tiles ahead
    struct Pages {
        int a, b, c, d;
        __device__ __forceinline__ int at(int u) const { return u == 0 ? a : u == 1 ? b : u == 2 ? c : d; }
        __device__ __forceinline__ uint32_t ok() const {   // a bit for each
            if (SRC != kPages) return 0xFFFFFFFFu;
            return 0xFFFFFFF0u | (uint32_t)(a >= 0) | (uint32_t)(b >= 0) << 1 | (uint32_t)(c >= 0) << 2 | (uint32_t)(d >= 0) << 3;
        }
    };
    auto pages_of = [&](int t) __attribute__((always_inline)) {
        Pages x{0, 0, 0, 0};
        if (SRC != kPages) return x;
        const int j0 = g.tile(i0 + max(min(t, n_tiles - 1), 0)) * BN;
        x.a = page_at(a, tab, j0);
        x.b = page_at(a, tab, j0 + 16);
        if (BN == 64) {
            x.c = page_at(a, tab, j0 + 32);
            x.d = page_at(a, tab, j0 + 48);
        }
        return x;
    };
    auto copy = [&](auto values, int t, const Pages &pages) __attribute__((always_inline)) {
        constexpr bool V = decltype(values)::value;
        const int j0 = g.tile(i0 + t) * BN;
        const bool every = whole_tile(pl, pf, j0);   // some row sees each of its keys
        const int ln = X::QL ? fresh_lane() : lane;
        uint32_t offs[2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int c = (n * W + w) * 64 + ln, r = c / CH, x = c % CH;
            offs[n] = (uint32_t)(ln / CH) * (V ? v_row : k_row) + 16 * (x ^ (V ? X::val_swz(r) : X::key_swz(r)));
        }
#pragma unroll
        for (int n = 0; n < COPIES; n++) {
            const int c0 = (n * W + w) * 64, r0 = c0 / CH;
            const int page = pages.at(r0 / 16);
            const uint32_t off = offs[V ? 0 : n & 1], to = base + (V ? 2 + (t & 1) : t & 1) * TENSOR + 16 * c0;
            const char *from;
            if (SRC == kPages) from = (V ? v_base : k_base) + (int64_t)max(page, 0) * page_bytes + ((j0 + r0) & page_mask) * (2 * D);
            else from = (V ? v_base : k_base) + (int64_t)(j0 + r0) * (V ? v_row : k_row);
            if (every && page >= 0) {
                dma16(from, off, to);
            } else {   // what no row sees counts for nothing, whatever lies there
                const int j = j0 + r0 + ln / CH;
                const bool use = page >= 0 && j <= pl && (!a.window || j > pf - a.window || j < a.sinks);
                dma16(use ? from + off : (const char *)kZeros, to);
            }
        }
    };
    const std::false_type keys;
    const std::true_type values;
    Pages now = pages_of(0), next = pages_of(1), after = pages_of(2), last;   // of tiles t .. t + 3
    if (n_tiles > 0) {
        copy(keys, 0, now);
        copy(values, 0, now);
    }
    if (n_tiles > 1) copy(keys, 1, next);
    if (tid == 0) *flag = 0;
    const uint32_t q_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)(marks + many_marks(D) + 16);
    X x;
    x.start((const R *)a.q + (it.s.start + tok) * a.q_tok + (it.head * a.G + rq - tok * a.G) * a.q_head, a.scale, q_lds, it.s);
    wait_vm<0>();
    lds_barrier();
    typename X::F s[NB];
    auto has_keys = [&](int t) __attribute__((always_inline)) { return R0 + M * w < n_rows && t < n_tiles && g.tile(i0 + t) * BN <= wl; };
    if (has_keys(0)) x.scores(base, s);

    auto vals_at = [&](int t) __attribute__((always_inline)) { return base + (2 + (t & 1)) * TENSOR; };
    auto keys_at = [&](int t) __attribute__((always_inline)) { return base + (t & 1) * TENSOR; };
    // Tile t's values and the next one's keys are there; what lies behind them is requested.
    auto turn = [&](int t) __attribute__((always_inline)) {
        last = pages_of(t + 3);
        wait_vm<0>();
        lds_barrier();
        if (t + 2 < n_tiles) copy(keys, t + 2, after);
        if (t + 1 < n_tiles) copy(values, t + 1, next);
    };
    auto advance = [&]() __attribute__((always_inline)) {
        now = next;
        next = after;
        after = last;
    };
    // Every row of the work-group sees all of tile t, and this wavefront some of the next.
    auto plain = [&](int t) __attribute__((always_inline)) {
        const int j0 = g.tile(i0 + t) * BN;
        return has_keys(t + 1) && whole_tile(pf, pl, j0) && now.ok() == 0xFFFFFFFFu;
    };
    auto any_tile = [&](int t) __attribute__((always_inline)) {
        const int j0 = g.tile(i0 + t) * BN;
        turn(t);
        const uint32_t page_ok = now.ok();
        bool spoilt = false;
        if (page_ok != 0xFFFFFFFFu || !whole_tile(pf, pl, j0)) {
            char *const vt = lds + (2 + (t & 1)) * TENSOR;
            if (X::find_spoilt(vt)) *flag = 1;
            lds_barrier();
            spoilt = __builtin_amdgcn_readfirstlane(*flag) != 0;
            if (spoilt) {
                lds_barrier();
                if (tid == 0) *flag = 0;
                X::mark_spoilt(vt, marks);
                lds_barrier();
            }
        }
        if (has_keys(t)) {
            const int p = it.s.pos0 + token_of(a, min(R0 + M * w + (X::QL ? fresh_lane() : lane) % M, n_rows - 1));
            uint32_t vis;
            const bool seen = x.look(a, p, j0, page_ok, vis);
            x.template raise<true>(s, vis, seen);
            x.template weigh<true>(vals_at(t), s, vis);
            if (spoilt) x.take_spoilt(a, p, j0, page_ok, marks);
        }
        if (has_keys(t + 1)) x.scores(keys_at(t + 1), s);
        advance();
    };
    // (Three loops, not one with two paths: the sums would be moved between the paths' registers at every tile.)
    int t = 0;
    for (; t < n_tiles && !plain(t); t++) any_tile(t);
    for (; t < n_tiles && plain(t); t++) {
        turn(t);
        x.template raise<false>(s, 0, true);
        x.template weigh<false>(vals_at(t), s, 0);
        x.scores(keys_at(t + 1), s);
        advance();
    }
    for (; t < n_tiles; t++) any_tile(t);
    const int last_row = R0 + M * w + (X::QL ? fresh_lane() : lane) % M;
    x.finish(a, it, last_row, token_of(a, min(last_row, n_rows - 1)));
}

// The same with keys and values that pass through registers: rows of any alignment, and floats in NK planes. A tile's values are put into LDS beside
// its scores, the next one's keys beside its sums, so that what makes planes of them runs beside the matrix cores; two barriers a tile. 2000 float rows of 16 heads on 4 of
// 256 in five prompts 148 us by the trace: 24 operand reads of 1 KB for 48 products of 16 clocks and about as many clocks of vector instructions, a work-group a CU.
template <int D, class E, int NP, int NK, int RT, int M>
__global__ __launch_bounds__(8192 / M, 2) void attn_many_any_kernel(const BatchAttnArgs a) {
    typedef typename Row<RT>::t R;
    typedef WaveRows<D, E, NP, NK, R, M> X;
    constexpr int BN = X::BN, NB = X::NB, CH = X::CH, TENSOR = X::TENSOR, PLANE = X::PLANE;
    constexpr int W = kManyRows / M, COPIES = BN * CH / (64 * W);   // wavefronts; pieces of 8 elements a lane and tensor
    extern __shared__ __align__(1024) char lds[];   // keys, values, marks, flag
    char *const vb = lds + TENSOR;
    uint8_t *const marks = (uint8_t *)lds + 2 * TENSOR;
    int *const flag = (int *)(marks + many_marks(D));
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    Item it;
    if (!find_item<kManyRows, BN, false>(a, blockIdx.x, it)) return;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const int R0 = it.tile * kManyRows, n_rows = it.s.rows * a.G;
    const int row = R0 + M * w + lane % M, rq = min(row, n_rows - 1), tok = token_of(a, rq), p = it.s.pos0 + tok;
    const int pf = it.s.pos0 + token_of(a, R0), pl = it.s.pos0 + token_of(a, min(R0 + kManyRows, n_rows) - 1);
    const int wl = it.s.pos0 + token_of(a, min(R0 + M * w + M, n_rows) - 1);
    const Range g = range_of<BN>(a, pf, pl);
    const int i0 = part_from(g.n, it.piece, it.pieces), n_tiles = part_from(g.n, it.piece + 1, it.pieces) - i0;
    Rows<R, 8> kx[COPIES], vx[COPIES];
    // (no branch about a load, and behind the last tile that one again: so it is known how many are on their way)
    auto request = [&](auto values, int t) __attribute__((always_inline)) {
        constexpr bool V = decltype(values)::value;
        const int j0 = g.tile(i0 + min(t, n_tiles - 1)) * BN;
#pragma unroll
        for (int n = 0; n < COPIES; n++) {
            const int c = n * 64 * W + tid, r = c / CH, e = c % CH, j = j0 + r;
            const R *const from = V ? (const R *)a.v + (it.s.start + j) * a.v_tok + it.head * a.v_head + 8 * e
                                    : (const R *)a.k + (it.s.start + j) * a.k_tok + it.head * a.k_head + 8 * e;
            const bool use = j <= pl && (!a.window || j > pf - a.window || j < a.sinks);   // what no row sees counts for nothing, whatever lies there
            (V ? vx[n] : kx[n]) = *(const __attribute__((address_space(1))) Rows<R, 8> *)(uintptr_t)(use ? from : (const R *)kZeros);
        }
    };
    auto put = [&](auto values) __attribute__((always_inline)) {
        constexpr bool V = decltype(values)::value;
#pragma unroll
        for (int n = 0; n < COPIES; n++) {
            const int c = n * 64 * W + tid, r = c / CH, e = c % CH;
            const Rows<R, 8> &x = V ? vx[n] : kx[n];
            V8<E> p[NK];
            if constexpr (NK == 1) {
                p[0] = __builtin_bit_cast(V8<E>, x);
            } else {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] = (float)x[i];
                planes<E, NK>(f, p);
            }
            char *const to = (V ? vb : lds) + 16 * (r * CH + (e ^ (V ? X::val_swz(r) : X::key_swz(r))));
#pragma unroll
            for (int k = 0; k < NK; k++) *(V8<E> *)(to + k * PLANE) = p[k];
        }
    };
    const std::false_type keys;
    const std::true_type values;
    if (n_tiles > 0) {
        request(keys, 0);
        request(values, 0);
    }
    if (tid == 0) *flag = 0;
    const uint32_t q_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)(marks + many_marks(D) + 16);
    X x;
    x.start((const R *)a.q + (it.s.start + tok) * a.q_tok + (it.head * a.G + rq - tok * a.G) * a.q_head, a.scale, q_lds, it.s);
    if (n_tiles > 0) {
        put(keys);
        request(keys, 1);
    }
    auto put_values = [&](int t) __attribute__((always_inline)) {
        put(values);
        request(values, t + 1);
    };
    auto put_keys = [&](int t) __attribute__((always_inline)) {   // the next tile's
        put(keys);
        request(keys, t + 2);
    };
    auto whole_tile = [&](int f, int l, int j0) __attribute__((always_inline)) { return j0 + BN - 1 <= f && (!a.window || j0 > l - a.window || j0 + BN - 1 < a.sinks); };
    auto plain = [&](int t) __attribute__((always_inline)) { return R0 + M * w < n_rows && whole_tile(pf, pl, g.tile(i0 + t) * BN); };
    auto any_tile = [&](int t) __attribute__((always_inline)) {
        const int j0 = g.tile(i0 + t) * BN;
        const bool here = R0 + M * w < n_rows && j0 <= wl;
        typename X::F s[NB];
        lds_barrier();
        if (here) x.scores(base, s);
        put_values(t);
        lds_barrier();
        bool spoilt = false;
        if (!whole_tile(pf, pl, j0)) {
            if (X::find_spoilt(vb)) *flag = 1;
            lds_barrier();
            spoilt = __builtin_amdgcn_readfirstlane(*flag) != 0;
            if (spoilt) {
                lds_barrier();
                if (tid == 0) *flag = 0;
                X::mark_spoilt(vb, marks);
                lds_barrier();
            }
        }
        if (here) {
            uint32_t vis;
            const bool seen = x.look(a, p, j0, 0xFFFFFFFFu, vis);
            x.template raise<true>(s, vis, seen);
            x.template weigh<true>(base + TENSOR, s, vis);
            if (spoilt) x.take_spoilt(a, p, j0, 0xFFFFFFFFu, marks);
        }
        put_keys(t);
    };
    const bool early = w >= W / 2;   // of a SIMD's two wavefronts one makes planes while the other has the matrix cores
    int t = 0;
    for (; t < n_tiles && !plain(t); t++) any_tile(t);
    for (; t < n_tiles && plain(t); t++) {
        typename X::F s[NB];
        lds_barrier();
        if (early) put_values(t);
        x.scores(base, s);
        if (!early) put_values(t);
        lds_barrier();
        if (early) put_keys(t);
        x.template raise<false>(s, 0, true);
        x.template weigh<false>(base + TENSOR, s, 0);
        if (!early) put_keys(t);
    }
    for (; t < n_tiles; t++) any_tile(t);
    x.finish(a, it, row, tok);
}

template <class F>
static int many_run(F *f, int threads, int bytes, const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    if (hipFuncSetAttribute((const void *)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return -1;
    f<<<dim3((unsigned)items), threads, bytes, st>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int D, class E, int NP, int RT, int SRC>
static int many(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    constexpr int M = NP == 1 ? 32 : 16;   // rows a wavefront (WaveRows)
    typedef WaveRows<D, E, NP, 1, typename Row<RT>::t, M> X;
    return many_run(attn_many_kernel<D, E, NP, RT, SRC, M>, 8192 / M, 4 * X::TENSOR + many_marks(D) + 16 + X::QL * 1024 * (kManyRows / M), a, items, st);
}
template <int D, class E, int NP, int NK, int RT>
static int many_any(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    constexpr int M = NP == 1 && D <= 128 ? 32 : 16;
    typedef WaveRows<D, E, NP, NK, typename Row<RT>::t, M> X;
    return many_run(attn_many_any_kernel<D, E, NP, NK, RT, M>, 8192 / M, 2 * X::TENSOR + many_marks(D) + 16 + X::QL * 1024 * (kManyRows / M), a, items, st);
}
template <int D>
static int many(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    if (a.table) {
        if (a.type == kRowF16) return many<D, _Float16, 1, kRowF16, kPages>(a, items, st);
        if (a.type == kRowBf16) return many<D, __bf16, 1, kRowBf16, kPages>(a, items, st);
        if (a.kv_type == kRowF16) return many<D, _Float16, 2, kRowF32, kPages>(a, items, st);
        return many<D, __bf16, 3, kRowF32, kPages>(a, items, st);
    }
    if (a.type == kRowF32) return many_any<D, __bf16, 3, 3, kRowF32>(a, items, st);
    // (a lane's offset within a copy, 8 rows at most, has 32 bits)
    const bool whole = !(((uintptr_t)a.k | (uintptr_t)a.v) & 15) && !((a.k_tok | a.k_head | a.v_tok | a.v_head) & 7) &&
                       a.k_tok >= 0 && a.v_tok >= 0 && std::max(a.k_tok, a.v_tok) < (1 << 27);
    if (a.type == kRowF16) {
        return whole ? many<D, _Float16, 1, kRowF16, kRows16>(a, items, st) : many_any<D, _Float16, 1, 1, kRowF16>(a, items, st);
    }
    return whole ? many<D, __bf16, 1, kRowBf16, kRows16>(a, items, st) : many_any<D, __bf16, 1, 1, kRowBf16>(a, items, st);
}
int attn_many_launch(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    return a.D == 64 ? many<64>(a, items, st) : a.D == 128 ? many<128>(a, items, st) : many<256>(a, items, st);
}

// ---------------------------------------------------------------- launch --

// How a batch is run: in one launch of the kernel for few rows or of that for many (only = 0), or in one of each, for the requests of up to
// kFewLimit rows a kv head (1) and for the others (2).
struct Run {
    int BM, only, target, least;
    int64_t tiles, items;   // row tiles times heads, and work items, at most
};
// Work-groups that the GPU's 256 CUs hold of the kernel at once.
static int held_of(const BatchAttnArgs &a, bool few) {
    return 256 * (few ? (a.D == 64 ? 3 : a.D == 128 && a.type != kRowF32 ? 2 : 1) : a.type == kRowF32 ? 1 : 2);
}
static Run run_of(const BatchAttnArgs &a, bool few, int only) {
    Run r;
    r.BM = few ? kFewRows : kManyRows;
    r.only = only;
    const int64_t rows = (int64_t)a.T * a.G, n = std::min<int64_t>(only == 2 ? std::min<int64_t>(a.n_req, rows / (kFewLimit + 1)) : a.n_req, a.T);
    r.tiles = rows / r.BM + n;
    if (only == 1) r.tiles = std::min(r.tiles, 2 * n);
    r.tiles *= a.Hkv;
    r.least = 8;
    const int held = held_of(a, few);
    const int BN = few ? kFewKeys : many_keys(a.D);
    const int64_t longest = ((a.table ? (int64_t)a.max_blocks << a.lg : a.T) + BN - 1) / BN;
    r.target = longest <= r.least ? 0 : held;   // pieces aimed at
    r.items = r.target ? std::min(r.tiles * ((longest + r.least - 1) / r.least), r.tiles + r.target) : r.tiles;
    return r;
}
static int runs_of(const BatchAttnArgs &a, Run (&r)[2]) {
    // Prompts in 16 bits whose tiles of 16 rows the GPU holds at once are faster in those too: 51 rows of 2 heads on 1 of 128 8.5 us, 12.7 in tiles of 128; 200 of
    // 32 on 8 14.8, 17.3, but 256 of them 30, 18.6.
    const bool few = a.table ? (int64_t)(a.max_new > 0 ? a.max_new : a.T) * a.G <= kFewLimit
                             : a.type != kRowF32 && a.T <= 1024 && ((int64_t)a.T * a.G / kFewRows + std::min(a.n_req, a.T)) * a.Hkv <= held_of(a, true);
    if (few || !a.table || a.n_req == 1) {
        r[0] = run_of(a, few, 0);
        return 1;
    }
    r[0] = run_of(a, true, 1);
    r[1] = run_of(a, false, 2);
    return 2;
}
// (Requests may be cut whatever the bounds of the call say: a batch of 8200 rows may be one prompt among a thousand empty ones, 2 heads on 1 of 128: 97 us, 204
// uncut; over pages one row may see more than all the others do, 100000 positions beside 103 requests of 100, 32 heads on 8 of 128: 101 us, 1298 uncut. A join that
// finds nothing costs 2 to 6 us.)
constexpr int kPer = 64;   // floats in front of the partials, whose rows begin at cache lines then: a.per
static int64_t slot_floats(const BatchAttnArgs &a, int BM) { return (int64_t)BM * (a.D + 2); }

int64_t batch_attn_part_floats(const BatchAttnArgs &a) {
    int64_t most = 0;
    for (const bool few : {true, false}) {   // a smaller batch may run in the other tiles
        if (few ? !a.table && a.type == kRowF32 : a.table && (int64_t)(a.max_new > 0 ? a.max_new : a.T) * a.G <= kFewLimit) continue;
        const Run r = run_of(a, few, 0);
        if (r.target) most = std::max(most, kPer + std::min<int64_t>(r.items, 2 * r.target) * slot_floats(a, r.BM));
    }
    return most;
}

int batch_attn_launch(const BatchAttnArgs &args, int64_t part_floats, hipStream_t st) {
    Run runs[2];
    const int n = runs_of(args, runs);
    for (int i = 0; i < n; i++) {
        const Run &r = runs[i];
        if (!r.tiles) continue;
        BatchAttnArgs a = args;
        a.only = r.only;
        a.slots = (int)std::min<int64_t>(std::max<int64_t>(part_floats - kPer, 0) / slot_floats(a, r.BM), 1 << 20);
        // 65 to 128 requests whose tiles the GPU holds at once sum for themselves side by side (66 to 100 of 2 heads on 1 of 128 12 to 20 us, 13.5 to 21.5 with the
        // launch; 200 prompts of 20 tokens 27 without, 19 with it).
        a.per = a.n_req > 128 || (a.n_req > 64 && r.tiles > 256) ? (int32_t *)args.part : nullptr;
        a.part = args.part + kPer;
        // at most 2 a.target items are in pieces
        a.target = a.slots >= std::min<int64_t>(r.items, 2 * r.target) ? r.target : std::min(r.target, a.slots / 2);
        a.least = r.least;
        if (a.target && a.per && attn_cut_launch(a, r.BM, st)) return -1;
        const int64_t items = a.target ? std::min(r.items, r.tiles + a.target) : r.tiles;
        if (r.BM == kFewRows ? attn_few_launch(a, items, st) : attn_many_launch(a, items, st)) return -1;
        if (a.target && attn_merge_launch(a, r.BM, std::min<int64_t>(r.tiles, a.target), r.tiles > 1024, st)) return -1;
    }
    return 0;
}

}  // namespace xjk
