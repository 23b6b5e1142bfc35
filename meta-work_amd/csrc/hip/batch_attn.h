// Attention over batches of requests of different lengths: what its kernels share (gfx950).
//
// The rows of a request and kv head are its new tokens times the G = H / Hkv query heads that read that kv head, row R being
// token R / G, query head R % G. A work item is a tile of BM rows of a request and a kv head over a piece of the key tiles
// (of BN positions) that they see. The kernels form S^T = K Q^T, so that a lane holds scores of one row only, and O^T = V^T P^T
// straight from them: with the keys of an instruction taken in the order in which the first product leaves them, the weights
// are the second one's operand as they are.
#pragma once
#include "common.h"
#include "kernels.h"

namespace xjk {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_u __attribute__((ext_vector_type(4), aligned(2)));   // rows of any 2-byte alignment
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8_u __attribute__((ext_vector_type(8), aligned(4)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// Operands of the matrix cores.
template <class E>
struct Op;
template <>
struct Op<_Float16> {
    typedef hf8 v8;
    static constexpr uint32_t kExp = 0x7C00, kOne = 0x3C00;
    // Weights are 2^lift p (lift_of) to a reference that the running maximum may exceed by kTol before the sums are rescaled to it (on random
    // scores nearly every tile raises some row's maximum a little), 2^15 at most: bits are lost from 2^-22 of the largest on only.
    static constexpr float kTol = 7.f;
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x16 mfma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Op<__bf16> {
    typedef bf8 v8;
    static constexpr uint32_t kExp = 0x7F80, kOne = 0x3F80;
    static constexpr float kTol = 8.f;
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x16 mfma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <class E>
using V8 = typename Op<E>::v8;

// Eight numbers as NP planes that add up to them: one plane rounds to nearest; f16 in two keeps 22 bits (of numbers scaled so that
// the planes are no subnormals); bf16 takes the leading 8 bits of what is left in each, 16 in two, all in three. (An infinity's further
// planes are NaN: a product with it is not finite.)
template <class E, int NP>
__device__ __forceinline__ void planes(const float (&x)[8], V8<E> (&p)[NP]) {
    if constexpr (NP == 1) {
#pragma unroll
        for (int i = 0; i < 8; i++) p[0][i] = (E)x[i];
    } else if constexpr (__is_same(E, _Float16)) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[0][i] = (E)x[i];
            p[1][i] = (E)(x[i] - (float)p[0][i]);
        }
    } else {
        uint32_t w[NP][4];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            uint32_t u[NP], v[NP];
            float a = x[i], b = x[i + 1];
#pragma unroll
            for (int k = 0; k < NP; k++) {
                u[k] = __float_as_uint(a) & 0xFFFF0000u;
                v[k] = __float_as_uint(b) & 0xFFFF0000u;
                a -= __uint_as_float(u[k]);
                b -= __uint_as_float(v[k]);
                w[k][i / 2] = __builtin_amdgcn_perm(v[k], u[k], 0x07060302u);
            }
        }
#pragma unroll
        for (int k = 0; k < NP; k++) p[k] = __builtin_bit_cast(V8<E>, u32x4{w[k][0], w[k][1], w[k][2], w[k][3]});
    }
}

// The larger of a lane's value and that of lane l ^ 16, l ^ 32.
__device__ __forceinline__ float max_x16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// x / G of a row x < 2^28.
__device__ __forceinline__ int token_of(const BatchAttnArgs &a, int x) {
    const int q = (int)__umulhi((uint32_t)x, a.inv_g);   // or one less
    return q + (x - q * a.G >= a.G);
}
constexpr int kFewRows = 16, kFewKeys = 32, kFewLimit = 2 * kFewRows;   // requests of up to kFewLimit rows a kv head are few
constexpr int kManyRows = 128;
constexpr int many_keys(int D) { return D == 256 ? 32 : 64; }
// The rows of one request.
struct Seq {
    int r, start, rows, pos0;   // its rows of q, the first one's position
    int tiles, len;             // row tiles; key tiles that the last of them sees
};
// The key tiles that rows at positions pf .. pl see: n of them, tile(i) the i-th.
struct Range {
    int first, n_sink, n;
    __device__ __forceinline__ int tile(int i) const { return i < n_sink ? i : first + i - n_sink; }
};
template <int BN>
__device__ __forceinline__ Range range_of(const BatchAttnArgs &a, int pf, int pl) {
    Range g{0, 0, 0};
    if (pl < 0) return g;
    if (a.window) {
        g.first = max(0, pf - a.window + 1) / BN;
        g.n_sink = min((min(a.sinks, pl + 1) + BN - 1) / BN, g.first);
    }
    g.n = g.n_sink + pl / BN - g.first + 1;
    return g;
}
template <int BM, int BN>
__device__ __forceinline__ Seq seq_of(const BatchAttnArgs &a, int r) {
    Seq s{};
    if (r >= a.n_req) return s;
    const int c0 = a.cu[r], c1 = a.cu[r + 1];
    s.r = r;
    s.start = min(max(c0, 0), a.T);
    s.rows = min(max(c1, s.start), a.T) - s.start;
    if (a.kv_len) s.pos0 = (int)max((int64_t)min(max(a.kv_len[r], 0), a.max_blocks << a.lg) - ((int64_t)c1 - c0), (int64_t)(-1 << 30));
    s.tiles = (s.rows * a.G + BM - 1) / BM;
    if (a.only && (a.only == 1) != (s.rows * a.G <= kFewLimit)) s.tiles = 0;
    if (s.tiles) s.len = range_of<BN>(a, s.pos0 + token_of(a, (s.tiles - 1) * BM), s.pos0 + s.rows - 1).n;
    return s;
}
__device__ __forceinline__ float wave_sum(float v) {   // the same for every lane and in the same order
    v = xjd::row16_sum(v);
    auto at = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
    return (at(0) + at(16)) + (at(32) + at(48));
}
// Part `piece` of n tiles in `pieces` parts.
__device__ __forceinline__ int part_from(int n, int piece, int pieces) {
    const int q = n / pieces;
    return q * piece + min(piece, n - q * pieces);
}
struct Item {
    Seq s;
    int tile, head, piece, pieces, slot;
};
// With U key tiles over all row tiles and heads, u * a.Hkv, a piece is about U / a.target of them and no fewer than a.least, so that the pieces are
// alike whatever the lengths. At most a.target + (row tiles * heads) items, 2 a.target of them in pieces: a request is cut only if it has
// more than a piece's tiles.
__device__ __forceinline__ int piece_of(const BatchAttnArgs &a, float u) { return max(a.least, (int)fminf(u * a.Hkv * 1.0001f / a.target, 1e9f) + 1); }
// Work item `item` (with MERGE: row tile and head `item` of those in more than one piece); false beyond the last. Every
// wavefront finds its own, from the lengths, 64 requests at a time, and the tiles of a piece too, if they are not in a.per. (Of more than 64 requests those of less
// than two pieces are not worth a cut: 5 rows of 200 requests of up to 2000 positions, 32 heads on 8 of 128: 103 us, 117 where some are cut.) Where the uncut items are at most half of a.target, what
// the GPU holds at once, longer pieces that it holds at once are better than the last of more (5 rows of 8 requests behind a window of
// 2048, 16 heads on 4 of 256: 256 items 30 us, 512 47).
template <int BM, int BN, bool MERGE>
__device__ __forceinline__ bool find_item(const BatchAttnArgs &a, int item, Item &it) {
#pragma clang fp contract(off)   // the kernels of a call cut alike
    const int lane = threadIdx.x & 63;
    int per = INT32_MAX;
    const bool once = a.n_req <= 64;
    Seq s{};
    if (once) s = seq_of<BM, BN>(a, lane);
    if (a.target && a.per) {
        per = __builtin_amdgcn_readfirstlane(*a.per);
        if (MERGE && per == INT32_MAX) return false;   // nothing is cut
    } else if (a.target && !once) {
        float u = 0.f;
        int most = 0;
        for (int r0 = 0; r0 < a.n_req; r0 += 64) {
            s = seq_of<BM, BN>(a, r0 + lane);
            u += (float)s.tiles * (float)s.len;
            most = max(most, s.len);
        }
        per = piece_of(a, wave_sum(u));
        if (!__any(most > 2 * per)) {
            if (MERGE) return false;
            per = INT32_MAX;
        }
    } else if (a.target) {
        per = piece_of(a, wave_sum((float)s.tiles * (float)s.len));
        const float uncut = wave_sum((float)s.tiles) * a.Hkv;
        for (int k = 0; k < 8 && 2.f * uncut <= (float)a.target; k++) {
            const float n = wave_sum((float)s.tiles * fmaxf(ceilf((float)s.len * __builtin_amdgcn_rcpf((float)per)), 1.f)) * a.Hkv;   // about
            if (n <= (float)a.target) break;
            per += max(1, per / 16);
        }
        if (MERGE && !__any(s.len > per)) return false;
    }
    if (BM == kManyRows && once && a.n_req > 1) {   // the requests that see most first: the last items are then short ones
        const int key = s.tiles ? s.len : -1;
        int rank = 0;
        for (int j = 0; j < a.n_req; j++) {
            const int other = __builtin_amdgcn_readlane(key, j);
            rank += other > key || (other == key && j < lane);
        }
        auto move = [&](int v) { return __builtin_amdgcn_ds_permute(4 * (lane < a.n_req ? rank : lane), v); };
        s = Seq{move(s.r), move(s.start), move(s.rows), move(s.pos0), move(s.tiles), move(s.len)};
    }
    int items = 0, slots = 0;
    for (int r0 = 0; r0 < a.n_req; r0 += 64) {
        if (!once) s = seq_of<BM, BN>(a, r0 + lane);
        const int pieces = s.len > per ? (int)((uint32_t)(s.len + per - 1) / (uint32_t)per) : 1, heads = s.tiles * a.Hkv;
        const int n_slot = pieces > 1 ? heads * pieces : 0, n = MERGE ? (pieces > 1 ? heads : 0) : heads * pieces;
        const int to = items + xjd::wave_scan(n), slot_to = slots + xjd::wave_scan(n_slot);
        const unsigned long long m = __ballot(to > item);
        if (m) {
            const int l = __builtin_ctzll(m);
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            it.s = Seq{get(s.r), get(s.start), get(s.rows), get(s.pos0), get(s.tiles), get(s.len)};
            it.pieces = get(pieces);
            const int local = item - get(to - n), slot = get(slot_to - n_slot);
            it.head = local % a.Hkv;
            const int q = local / a.Hkv;
            it.piece = MERGE ? 0 : q % it.pieces;
            const int i = MERGE ? q : q / it.pieces;
            it.tile = it.s.tiles - 1 - i;   // those that see most first
            it.slot = slot + (i * it.pieces + it.piece) * a.Hkv + it.head;   // the next piece's is Hkv further
            return true;
        }
        items = __builtin_amdgcn_readlane(to, 63);
        slots = __builtin_amdgcn_readlane(slot_to, 63);
    }
    return false;
}

// A page of the request's row for position j, uniform over the wavefront, or -1. (Read as a constant: a vector load would be
// waited for behind the keys and values on their way.)
__device__ __forceinline__ int page_at(const BatchAttnArgs &a, const int32_t *row, int j) {
    const int b = __builtin_amdgcn_readfirstlane(j) >> a.lg;
    const int p = b < a.max_blocks ? ((const __attribute__((address_space(4))) int32_t *)row)[b] : -1;
    return p >= 0 && p < a.n_pages ? p : -1;
}
__device__ __forceinline__ bool sees(const BatchAttnArgs &a, int p, int j) {
    return j <= p && (!a.window || j > p - a.window || j < a.sinks);
}

// The power of two by which a request's weights are raised. Over f16 values no sum leaves fp32's range. bf16's range is fp32's: a weight is
// 2^-n at most, where the request sees up to 2^n positions, so that no sum of weighted values is beyond the largest of them. (Small values pay for it: a
// sum has 24 bits from 2^(n - 93) on, of 16000 positions from 2^-79.)
template <class E, int BN>
__device__ __forceinline__ float lift_of(const Seq &s) {
    if constexpr (__is_same(E, _Float16)) return 8.f;
    return -(Op<E>::kTol + (32 - __builtin_clz(max(s.len * BN, 2) - 1)));
}

// State of the splits in the work area: [slots][BM][D] unscaled sums, then [slots][BM] of (the largest score in powers of two,
// the weights' sum). A row that has seen nothing yet has the largest score -infinity.
__device__ __forceinline__ float *part_sums(const BatchAttnArgs &a, int64_t row, int D) { return a.part + row * D; }
__device__ __forceinline__ float2 *part_stat(const BatchAttnArgs &a, int64_t row, int BM, int D) {
    return (float2 *)(a.part + (int64_t)a.slots * BM * D) + row;
}

template <int RT>
struct Row;
template <>
struct Row<kRowF32> {
    typedef float t;
};
template <>
struct Row<kRowF16> {
    typedef _Float16 t;
};
template <>
struct Row<kRowBf16> {
    typedef __bf16 t;
};

// N elements of rows of any alignment.
template <class R, int N>
using Rows = R __attribute__((ext_vector_type(N), aligned(sizeof(R))));
// 1 / (1 + e^-g), for rows of 16 bits to 2^-20.
template <class R>
__device__ __forceinline__ float gate_of(float g) {
    if constexpr (sizeof(R) == 4) return xjd::sigm(g);
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f));
}
// Four finished elements of a row: y times 1 / l, through the gate.
template <class R>
__device__ __forceinline__ void finish4(f32x4 y, float inv, const R *gate, R *out) {
    Rows<R, 4> z;
    y *= inv;
    if (gate) {
        const Rows<R, 4> g = *(const Rows<R, 4> *)gate;
#pragma unroll
        for (int k = 0; k < 4; k++) y[k] *= gate_of<R>((float)g[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) z[k] = (R)y[k];
    *(Rows<R, 4> *)out = z;
}

// Scores that underflow every weight still count as seen: the running maximum (in powers of two, rounded up) stays finite.
constexpr float kLowest = -1e38f;

int attn_cut_launch(const BatchAttnArgs &a, int BM, hipStream_t st);
int attn_merge_launch(const BatchAttnArgs &a, int BM, int64_t groups, bool rare, hipStream_t st);
int attn_few_launch(const BatchAttnArgs &a, int64_t items, hipStream_t st);
int attn_many_launch(const BatchAttnArgs &a, int64_t items, hipStream_t st);

}  // namespace xjk
