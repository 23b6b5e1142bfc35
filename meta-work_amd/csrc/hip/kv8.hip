// A key/value cache in 8 bits with one scale per block of tokens and kv head,
// and grouped-query attention over it (gfx950): xjh_kv8_store, xjh_kv8_load,
// xjh_attn_kv8.
//
// A tile is 64 positions of a kv head, 64 D bytes of keys and as many of values, both
// cut into 1 KB units that one wavefront reads with 16 bytes per lane and has as
// matrix operands at once (lane l: li = l & 15, kq = l >> 4):
//   keys    unit (u, s): lane l holds key 16 u + li, dims 64 s + 16 kq .. + 15
//   values  unit (d): lane l holds dim 16 d + li of the keys 16 u + 4 kq + r, byte 4 u + r
// The scores S^T = K Q^T leave lane l with the keys 16 u + 4 kq + r of query row li,
// which are the weights that it multiplies with those values.
#include "common.h"
#include "kernels.h"
#include <algorithm>
#include <type_traits>

namespace xjk {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf4 __attribute__((ext_vector_type(4)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));   // rows of any 4-byte alignment

__device__ __forceinline__ int clamp_past(int npast, const int32_t *dev) {
    return dev ? min(max(*dev, 0), npast) : npast;
}

// ------------------------------------------------------------ quantising --

// Largest magnitude that counts for a scale.
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;   // NaN compares false
}
template <bool E4>
__device__ __forceinline__ float block_scale(float amax) {
    if (!(amax > 0.f)) return 0.f;
    float s;
    if constexpr (E4) {
        int e;
        const float m = frexpf(amax, &e);   // 448 = 0.875 * 2^9
        s = ldexpf(1.f, e - (m <= 0.875f ? 9 : 8));
    } else {
        s = (float)((double)amax / 127.0);   // 24 + 53 bits: rounded once
    }
    return fmaxf(s, 0x1p-126f);
}
// The codes of four values: nearest to the exact quotients x / s, ties to even (inv = 1 / s, 0 for s = 0).
//   e4m3: s is a power of two, the product with 1 / s is exact and converts to nearest even.
//   int8: the product, rounded by adding 1.5 * 2^23 (the sum's low byte is the code), is off by less than 2^-14. Where one lies
//   nearer than that to a border (one value in 8000), the rests decide: x - c s is exact in one fma (it is below s
//   and a multiple of the smaller ulp), and twice it is compared with s (s / 2 is no float where s is below 2^-125 and odd).
// FIN: they are finite, so no quotient is beyond the largest code by more than its rounding.
template <bool E4, bool FIN>
__device__ __forceinline__ uint32_t codes_of(const f32x4 x, float s, float inv) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        y[i] = x[i] * inv;
        if (FIN) continue;
        y[i] = y[i] != y[i] ? 0.f : y[i];   // NaN, and an infinity in a block of scale 0
        y[i] = __builtin_amdgcn_fmed3f(y[i], E4 ? -448.f : -127.f, E4 ? 448.f : 127.f);
    }
    if constexpr (E4) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    } else {
        constexpr float kMagic = 12582912.f;
        float r[4], far = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            r[i] = y[i] + kMagic;
            far = fmaxf(far, fabsf(y[i] - (r[i] - kMagic)));
        }
        if (__any(far > 0.5f - 0x1p-14f)) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float c = r[i] - kMagic;
                const float rest = fmaf(-c, s, x[i]), twice = rest + rest;
                const bool odd = (int)c & 1;
                if (twice > s || (twice == s && odd)) c += 1.f;
                else if (twice < -s || (twice == -s && odd)) c -= 1.f;
                r[i] = fminf(fmaxf(c, -127.f), 127.f) + kMagic;   // (an infinity's rest is one)
            }
        }
        const uint32_t u = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x0c0c0400u);
        return __builtin_amdgcn_perm(__float_as_uint(r[3]), __float_as_uint(r[2]), 0x04000c0cu) | u;
    }
}
// A code of scale s_old at the larger scale s: the quotient of the code's value
// (31 bits at most) by s in double is never on the wrong side of a border.
template <bool E4>
__device__ __forceinline__ uint32_t recode(uint32_t c, float s_old, float s) {
    if constexpr (E4) {
        const float y = __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * (s_old / s);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xFFu;
    } else {
        return (uint32_t)(int)rint((double)(int8_t)c * (double)s_old / (double)s) & 0xFFu;
    }
}
template <bool E4>
__device__ __forceinline__ float value_of(uint32_t c, float s) {
    if constexpr (E4) return __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * s;
    else return (float)(int8_t)c * s;
}

// Store and load move a tile in 8 groups of 8 positions by D / 4 lanes, a lane 4 dims, so that the float rows
// (four times the codes' bytes) go 16 bytes per lane and whole rows per instruction. Group q of the keys is 8
// positions in a row; of the values the positions 16 u + 4 (q / 2) + r with u / 2 = q % 2, whose codes of a dim are 8 bytes.
template <bool VAL>
__device__ __forceinline__ int group_pos(int q, int i) { return VAL ? 16 * (2 * (q & 1) + (i >> 2)) + 4 * (q >> 1) + (i & 3) : 8 * q + i; }

// 4 x 4 bytes turned: byte c of w[r] becomes byte r of the result's c.
__device__ __forceinline__ void turn4(const uint32_t (&w)[4], uint32_t (&v)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    v[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    v[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    v[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    v[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}
// The lane's codes: w[i] byte c = dim d0 + c of the group's position i.
template <int D, bool VAL>
__device__ __forceinline__ void get_codes(const uint8_t *tile, int q, int d0, uint32_t (&w)[8]) {
    if constexpr (VAL) {
        const uint8_t *p = tile + (d0 >> 4) * 1024 + (q >> 1) * 256 + (d0 & 15) * 16 + 8 * (q & 1);
        uint2 v[4];
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = *(const uint2 *)(p + 16 * c);
        const uint32_t x[4] = {v[0].x, v[1].x, v[2].x, v[3].x}, y[4] = {v[0].y, v[1].y, v[2].y, v[3].y};
        uint32_t lo[4], hi[4];
        turn4(x, lo);
        turn4(y, hi);
#pragma unroll
        for (int r = 0; r < 4; r++) w[r] = lo[r], w[4 + r] = hi[r];
    } else {
        const uint8_t *p = tile + (q >> 1) * (16 * D) + (d0 >> 6) * 1024 + ((d0 >> 4) & 3) * 256 + (q & 1) * 128 + (d0 & 15);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = *(const uint32_t *)(p + 16 * i);
    }
}
template <int D, bool VAL>
__device__ __forceinline__ void put_codes(uint8_t *tile, int q, int d0, const uint32_t (&w)[8]) {
    if constexpr (VAL) {
        uint8_t *p = tile + (d0 >> 4) * 1024 + (q >> 1) * 256 + (d0 & 15) * 16 + 8 * (q & 1);
        const uint32_t x[4] = {w[0], w[1], w[2], w[3]}, y[4] = {w[4], w[5], w[6], w[7]};
        uint32_t lo[4], hi[4];
        turn4(x, lo);
        turn4(y, hi);
#pragma unroll
        for (int c = 0; c < 4; c++) *(uint2 *)(p + 16 * c) = uint2{lo[c], hi[c]};
    } else {
        uint8_t *p = tile + (q >> 1) * (16 * D) + (d0 >> 6) * 1024 + ((d0 >> 4) & 3) * 256 + (q & 1) * 128 + (d0 & 15);
#pragma unroll
        for (int i = 0; i < 8; i++) *(uint32_t *)(p + 16 * i) = w[i];
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
// The largest of D / 4 consecutive lanes, in each of them. (Magnitudes as their bits: an instruction a step, where floats need
// one more to make a NaN quiet.)
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
template <int D>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(v))));
    if (D >= 128) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max((uint32_t)r[0], (uint32_t)r[1]);
    }
    if (D >= 256) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max((uint32_t)r[0], (uint32_t)r[1]);
    }
    return v;
}

// A work-group stores one tile of a kv head's keys or values (2 D threads, a group each D / 4): the
// rows' largest magnitudes, joined over every block in LDS, the scales, the codes. In a
// tile that is not new from end to end the codes of the other positions are read
// and written back as they are, those of a begun block at its new scale if that grew.
// A thread's 32 values are in flight at once; then it is vector instructions, some 400 in each of two wavefronts a SIMD: 2048
// rows of 4 heads of 256 in e4m3, 17 MB in and 4 out, 8.9 us (10.4 with the checks for values that are not finite at every
// one of them, now only in wavefronts that have some, and a division by the scale in every thread), one row 5.0.
template <int D, bool E4, bool VAL>
__device__ __forceinline__ void store_tile(const Kv8StoreArgs &a, float (*sm)[64]) {
    const int g = blockIdx.y, tid = threadIdx.x, q = tid / (D / 4), d0 = tid % (D / 4) * 4, B = 1 << a.c.lg;
    const int np = clamp_past(a.npast, a.npast_dev), kt = (np >> 6) + blockIdx.x, j0 = kt * 64, end = np + a.T;
    if (j0 >= end) return;
    const float *x = (VAL ? a.v : a.k) + g * D + d0;
    const int64_t tok = VAL ? a.v_tok : a.k_tok;
    uint8_t *tile = (VAL ? a.c.v : a.c.k) + ((int64_t)g * a.c.n_tiles + kt) * 64 * D;
    float *sp = (VAL ? a.c.vs : a.c.ks) + ((((int64_t)g * a.c.n_tiles + kt) * 64) >> a.c.lg);
    const bool whole = j0 >= np && j0 + 64 <= end;
    uint32_t w[8], m[8], top = 0;
    const float old_s = !whole && tid < 64 ? sp[tid >> a.c.lg] : 0.f;
    if (!whole) get_codes<D, VAL>(tile, q, d0, w);
    f32x4 y[8];
    bool any = whole;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int p = j0 + group_pos<VAL>(q, i);
        y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p >= np && p < end) any = true, y[i] = *(const f32x4_u *)(x + (int64_t)(p - np) * tok);
    }
    any = __any(any);   // else nothing of the wavefront's rows is new
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const u32x4 b = __builtin_bit_cast(u32x4, y[i]) & 0x7FFFFFFFu;
        m[i] = max(max(b.x, b.y), max(b.z, b.w));
        top = max(top, m[i]);
    }
    const bool fin = !__any(top >= 0x7F800000u);
    if (!fin)
#pragma unroll
        for (int i = 0; i < 8; i++)
            m[i] = __float_as_uint(fmaxf(fmaxf(finite_abs(y[i].x), finite_abs(y[i].y)), fmaxf(finite_abs(y[i].z), finite_abs(y[i].w))));
    if (any)
#pragma unroll
        for (int i = 0; i < 8; i++) m[i] = row_max<D>(m[i]);
    if (d0 == 0)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
            *(f32x4 *)&sm[0][group_pos<VAL>(q, i)] = f32x4{__uint_as_float(m[i]), __uint_as_float(m[i + 1]), __uint_as_float(m[i + 2]), __uint_as_float(m[i + 3])};
    __syncthreads();
    if (tid < 64) {   // position j0 + tid: sm[0] its block's scale, sm[1] the block's earlier scale if it is begun, sm[2] 1 / scale
        float t = sm[0][tid];
        for (int o = 1; o < B; o <<= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
        const int first = (j0 + tid) & -B;
        float s = block_scale<E4>(t), old = 0.f;
        if (first < np && first + B > np) {
            old = old_s;
            s = fmaxf(s, old);
        }
        sm[0][tid] = s;
        sm[1][tid] = old;
        sm[2][tid] = s > 0.f ? 1.f / s : 0.f;
        if ((tid & (B - 1)) == 0 && first < end && first + B > np) sp[tid >> a.c.lg] = s;
    }
    __syncthreads();
    auto code = [&](auto finite) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int pl = group_pos<VAL>(q, i), p = j0 + pl;
            if (whole || (p >= np && p < end)) w[i] = codes_of<E4, decltype(finite)::value>(y[i], sm[0][pl], sm[2][pl]);
        }
    };
    if (any) {
        if (fin) code(std::true_type{});
        else code(std::false_type{});
    }
    if (!whole)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int pl = group_pos<VAL>(q, i), p = j0 + pl;
            const float s = sm[0][pl], old = sm[1][pl];
            if (p < np && (p | (B - 1)) >= np && s > old)
                w[i] = recode<E4>(w[i] & 0xFFu, old, s) | recode<E4>(w[i] >> 8 & 0xFFu, old, s) << 8 |
                       recode<E4>(w[i] >> 16 & 0xFFu, old, s) << 16 | recode<E4>(w[i] >> 24, old, s) << 24;
        }
    put_codes<D, VAL>(tile, q, d0, w);
}
template <int D, bool E4>
__global__ __launch_bounds__(2 * D) void kv8_store_kernel(const Kv8StoreArgs a) {
    __shared__ __align__(16) float sm[3][64];
    if (blockIdx.z) store_tile<D, E4, true>(a, sm);
    else store_tile<D, E4, false>(a, sm);
}

// Read back, Y groups a thread. Bound by the rows that it writes: 32000 positions of 4 heads of 256, 66 MB in and 262 out, 65 us
// (5.0 TB/s); a few by the launch and one round trip (77 positions of one head of 128 3.1 us).
template <int D, bool E4, bool VAL, int Y>
__device__ __forceinline__ void load_tile(const Kv8LoadArgs &a) {
    const int g = blockIdx.y, tid = threadIdx.x, q = Y * (tid / (D / 4)), d0 = tid % (D / 4) * 4;
    const int kt = (a.pos0 >> 6) + blockIdx.x, j0 = kt * 64;
    const float *sp = (VAL ? a.c.vs : a.c.ks) + ((((int64_t)g * a.c.n_tiles + kt) * 64) >> a.c.lg);
    const uint8_t *tile = (VAL ? a.c.v : a.c.k) + ((int64_t)g * a.c.n_tiles + kt) * 64 * D;
    uint32_t w[Y][8];
#pragma unroll
    for (int y = 0; y < Y; y++) get_codes<D, VAL>(tile, q + y, d0, w[y]);
    float *out = (VAL ? a.v : a.k) + g * D + d0;
    const int64_t tok = VAL ? a.v_tok : a.k_tok;
#pragma unroll
    for (int y = 0; y < Y; y++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int pl = group_pos<VAL>(q + y, i), t = j0 + pl - a.pos0;
            if (t < 0 || t >= a.n) continue;
            const float s = sp[pl >> a.c.lg];
            *(f32x4_u *)(out + t * tok) = f32x4{value_of<E4>(w[y][i] & 0xFFu, s), value_of<E4>(w[y][i] >> 8 & 0xFFu, s),
                                                value_of<E4>(w[y][i] >> 16 & 0xFFu, s), value_of<E4>(w[y][i] >> 24, s)};
        }
}
template <int D, bool E4, int Y>
__global__ __launch_bounds__(2 * D / Y) void kv8_load_kernel(const Kv8LoadArgs a) {
    if (a.k && !(a.v && blockIdx.z)) load_tile<D, E4, false, Y>(a);
    else load_tile<D, E4, true, Y>(a);
}

// ------------------------------------------------------------- attention --

__device__ __forceinline__ f32x4 mfma16(hf8 a, hf8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Four codes to f16, exactly. int8: c + 128 in the low bits of 1024 is 1152 + c.
template <bool E4>
__device__ __forceinline__ void to_half4(uint32_t w, hf2 &x, hf2 &y) {
    if constexpr (E4) {
        x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
        y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    } else {
        const uint32_t b = w ^ 0x80808080u;
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), v = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
        hf2 p, q;
        __builtin_memcpy(&p, &u, 4);
        __builtin_memcpy(&q, &v, 4);
        const hf2 off = {(_Float16)1152.f, (_Float16)1152.f};
        x = p - off;
        y = q - off;
    }
}
__device__ __forceinline__ hf8 join8(hf2 a, hf2 b, hf2 c, hf2 d) { return hf8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; }
// 8 codes as an operand.
template <bool E4>
__device__ __forceinline__ hf8 to_half(uint32_t w0, uint32_t w1) {
    hf2 h[4];
    to_half4<E4>(w0, h[0], h[1]);
    to_half4<E4>(w1, h[2], h[3]);
    return join8(h[0], h[1], h[2], h[3]);
}

// Two values as f16 planes, y = hi + lo to 22 bits. y is opaque to the compiler: as the product that it
// comes from, it would be rounded to f16 in one step for hi and in two for lo, and where
// the two differ (one product in 8000) lo would miss a whole step of hi.
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split2(float y0, float y1, hf2 &hi, hf2 &lo) {
    asm("" : "+v"(y0), "+v"(y1));
    hi = __builtin_convertvector(f32x2{y0, y1}, hf2);
    lo = __builtin_convertvector(f32x2{fmaf((float)hi.x, -1.f, y0), fmaf((float)hi.y, -1.f, y1)}, hf2);   // (exact differences, one mixed fma each)
}

// The tiles that the tokens at p0 .. p1 see: the first ns (of the tokens that stay
// visible), then those from f on; n in all.
struct Tiles {
    int ns, f, n;
};
__host__ __device__ __forceinline__ Tiles tiles_of(int p0, int p1, int window, int sinks) {
    const int lo = window && p0 - window + 1 > 0 ? p0 - window + 1 : 0;
    Tiles t;
    t.f = lo >> 6;
    const int s = window ? (int)(((int64_t)sinks + 63) >> 6) : 0;
    t.ns = s < t.f ? s : t.f;
    t.n = t.ns + (p1 >> 6) - t.f + 1;
    return t;
}

// Softmax state in powers of two. With t = score + log2(value scale), the weights are
// kept relative to a reference M that is at least max t - kGrow: w = 2^(t - M) <= 2^kGrow
// enters as two f16 planes of w * kP (22 bits), whatever the scales' range: the term 2 * 2^(score - M), of which the total is the
// sum, times the value scale times kP / 2 (the largest scale, 2^128 / 127, times kP would be infinite). The sums are rescaled only
// when max t passes M by more than kGrow.
// A score is a sum of codes by queries, times what the queries were divided by over kK, times the key's scale times kK (2^127 at most, so
// that the product before it is as small as can be): no step is beyond float's range where the score is well within it. It is
// rounded before M is formed of it: one of 2^24 and more then lies on the grid that M has, and the largest's term is still near 1 (with an
// exact product in the sums, M's rounding alone would be a power of two; plus() keeps the compiler from that).
__device__ __forceinline__ float plus(float a, float b) {
#pragma clang fp contract(off)
    return a + b;
}
constexpr float kGrow = 8.f, kP = 128.f, kK = 64.f;
// 2^(2 x), to the smallest denormal: the exponential instruction leaves out what is below 2^-126, which beside value scales of 2^100 and
// more are the terms of all but a row's best keys (2^-149 is 2^-28 of the smallest total). One product more for 1 ulp more.
__device__ __forceinline__ float exp2_twice(float x) {
    const float h = __builtin_amdgcn_exp2f(x);
    return h * h;
}

// Work-group barrier ordering LDS accesses only (global loads in flight stay in flight).
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// The sum over the lanes l and l ^ 8 (a row of 16 turned by half).
__device__ __forceinline__ float add_ror8(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
}

// Some row at the positions p0 .. p1 does not see the whole tile at j0.
__device__ __forceinline__ bool tile_edge(const Kv8AttnArgs &a, int j0, int p0, int p1) {
    return j0 + 63 > p0 || (a.window && j0 <= p1 - a.window && j0 + 63 >= a.sinks);
}
// Positions j that no row of the work-group sees may never have been stored: they have no scale, and where their e4m3 codes
// are NaN a weight of 0 does not take them out. Those after `last`, the call's last token, and from `sinks` up to `lo`, where
// the first row's window begins (0 without).
__device__ __forceinline__ bool held(int j, int sinks, int lo, int last) { return j <= last && (j >= lo || j < sinks); }
// Not every position of the tile at j0 is held; the lane's bytes of one of its values units that are.
__device__ __forceinline__ bool tile_part(int j0, int sinks, int lo, int last) { return j0 + 63 > last || (j0 < lo && j0 + 63 >= sinks); }
__device__ __forceinline__ u32x4 held_bytes(int j0, int sinks, int lo, int last) {
    const int kq = (threadIdx.x & 63) >> 4;
    u32x4 m;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        m[u] = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) m[u] |= held(j0 + 16 * u + 4 * kq + r, sinks, lo, last) ? 0xFFu << (8 * r) : 0u;
    }
    return m;
}

// N units of 1 KB from p (uniform): a scalar base per 4 KB and one lane offset, so the addresses take no registers.
template <int N>
__device__ __forceinline__ void load_units(const uint8_t *p, uint32_t lane, u32x4 (&r)[N]) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {   // (N a power of two)
        auto b = (const __attribute__((address_space(1))) uint8_t *)(p + c * 1024);
        asm("" : "+s"(b));
#pragma unroll
        for (int i = 0; i < (N < 4 ? N : 4); i++) r[c + i] = *(const __attribute__((address_space(1))) u32x4 *)(b + lane + i * 1024);
    }
}

// sigmoid by the exponential and reciprocal instructions (1 ulp each).
__device__ __forceinline__ float sigm_fast(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * x)); }

// N groups of 4 sums, 16 dims apart from dim d0, of a row with reference M and total: the split's partial sums [row][split][M,
// total, -, -, D sums], or, unsplit, over the total and gated into the output row.
template <int N, int D = 64 * N>
__device__ __forceinline__ void finish(const Kv8AttnArgs &a, int g, int row, int sp, int d0, float M, float total, const f32x4 *o) {
    const int G = a.H / a.c.Hkv;
    if (a.n_split > 1) {
        float *part = a.part + (((int64_t)g * a.T * G + row) * a.n_split + sp) * (D + 4);
        if (d0 == 0) part[0] = M, part[1] = total;
#pragma unroll
        for (int i = 0; i < N; i++) *(f32x4 *)(part + 4 + d0 + 16 * i) = o[i];
        return;
    }
    const int t = row / G, h = g * G + row % G;
    const float inv = (2.f / kP) / total;
    float *op = a.out + t * a.o_tok + (int64_t)h * D + d0;
    f32x4 x[N];
    if (a.gate)
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = *(const f32x4_u *)(a.gate + t * a.g_tok + h * a.g_head + d0 + 16 * i);
#pragma unroll
    for (int i = 0; i < N; i++) {
        f32x4 v = o[i] * inv;
        if (a.gate)
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] *= sigm_fast(x[i][r]);
        *(f32x4_u *)(op + 16 * i) = v;
    }
}

// Attention of 8 or 16 rows (row = token * G + head of the kv head): a work-group takes R of them and a split of the tiles. Its
// four wavefronts share every tile, each a part of every step, so nothing is converted or summed twice and one tile (a
// short context's) takes a quarter of the time:
//   scores   16 keys each: K units from the cache to registers, the queries stay in registers
//   weights  a quarter of the (row, key) pairs each: scores and weights pass through LDS (a few KB a tile)
//   sums     a quarter of the dims each
// A wavefront's part of the next tile (8 KB at D = 256) is always in flight, two work-groups or more share a CU: a long cache
// streams (one token at 131000 positions, 16 heads on 4 of 256 dims: 268 MB in 48.8 us, 5.5 TB/s; a 1 GiB copy reaches 5.15). A short
// one is bound by latency: 4000 positions, 8.4 MB, 5.8 us, most of it the first loads and the way of a tile through the steps.
// A: tiles requested ahead of the one in use.
// An operand has 16 columns. R = 8: both planes of 8 rows, so a product costs one instruction; R = 16: one plane after the
// other.
template <int D, bool E4, int R, int A>
__global__ __launch_bounds__(256, 2) void kv8_attn_kernel(const Kv8AttnArgs a) {
    constexpr int NS = D / 64, NV = D / 64, NQ = 2 * NS;   // a wavefront's units of keys and of values; 32-dim steps of a score
    constexpr bool ST = R == 8;
    constexpr int NP = ST ? 1 : 2;                         // operands a step
    constexpr int QW = NQ >= 4 ? NQ / 4 : 1;               // steps whose queries a wavefront prepares
    __shared__ __align__(16) hf8 qs[NQ][NP][64];
    __shared__ __align__(16) f32x4 sb[4][64];          // scores [16 keys][lane]
    __shared__ __align__(16) uint8_t pb[2][NP][1024];  // weights as operands [32 keys][plane][lane]
    __shared__ __align__(16) float sc[2][3][64];       // [tile parity] scales of the keys times kK, of the values times kP / 2, their log2
    __shared__ float alb[16], mx[4][16];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, li = l & 15, kq = l >> 4;
    const int G = a.H / a.c.Hkv, rows = a.T * G, np = clamp_past(a.npast, a.npast_dev);
    const int g = blockIdx.x % a.c.Hkv, sp = blockIdx.y, r0 = (int)blockIdx.x / a.c.Hkv * R;
    const int p0 = np + r0 / G, p1 = np + min(r0 + R - 1, rows - 1) / G, last = np + a.T - 1;
    const int lo = a.window ? max(p0 - a.window + 1, 0) : 0;
    const Tiles tl = tiles_of(p0, p1, a.window, a.sinks);
    const int i0 = sp * a.per_split, i1 = min(i0 + a.per_split, tl.n);
    if (i0 >= tl.n) return;
    const uint8_t *kc = a.c.k + (int64_t)g * a.c.n_tiles * 64 * D + w * NS * 1024, *vc = a.c.v + (int64_t)g * a.c.n_tiles * 64 * D + w * NV * 1024;
    const int64_t s0 = ((int64_t)g * a.c.n_tiles * 64) >> a.c.lg;
    u32x4 kr[A][NS], vr[A][NV];
    float s1[A] = {};   // wavefront 0: the keys' scale of position l; 1: the values'
    auto tile = [&](int i) { return i < tl.ns ? i : tl.f + i - tl.ns; };
    auto load_k = [&](int kt, u32x4 (&kr)[NS], float &s1) {
        load_units<NS>(kc + (int64_t)kt * 64 * D, l * 16, kr);
        const int j = kt * 64 + l;
        if (w < 2) s1 = held(j, a.sinks, lo, last) ? (w ? a.c.vs : a.c.ks)[s0 + (j >> a.c.lg)] : 0.f;
    };
    auto load_v = [&](int kt, u32x4 (&vr)[NV]) { load_units<NV>(vc + (int64_t)kt * 64 * D, l * 16, vr); };
    load_k(tile(i0), kr[0], s1[0]);
    load_v(tile(i0), vr[0]);
    auto ahead = [&](int i) { return tile(A > 1 ? min(i + A, i1 - 1) : i + A); };   // (past the end: the last one again, so that the waits know how many are in flight)
    if constexpr (A > 1) {
        load_k(ahead(i0 - 1), kr[A - 1], s1[A - 1]);
        load_v(ahead(i0 - 1), vr[A - 1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int row = r0 + (li & (R - 1)), rq = min(row, rows - 1), t = rq / G, h = g * G + rq % G, pos = np + t;
    // the queries as operands, step i = 2 s + e the dims 64 s + 16 kq + 8 e .. + 7, x 2^-e = hi + lo, e per row
    float qsc;
    {
        const bool mine = w * QW < NQ;
        const float *qp = a.q + t * a.q_tok + h * a.q_head + 16 * kq;
        f32x4 x[QW][2];
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < QW; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int st = mine ? w * QW + i : 0;
                x[i][e] = *(const f32x4_u *)(qp + 64 * (st >> 1) + 8 * (st & 1) + 4 * e);
#pragma unroll
                for (int r = 0; r < 4; r++) m = fmaxf(m, fabsf(x[i][e][r]));
            }
        m = max_x16(max_x32(m));
        if (l < 16) mx[w][l] = m;
        lds_barrier();
        m = fmaxf(fmaxf(mx[0][li], mx[1][li]), fmaxf(mx[2][li], mx[3][li]));
        int e = 0;
        if (m < INFINITY) (void)frexpf(m, &e);   // m < 2^e
        e = max(e, -102) - 14;
        qsc = ldexpf(a.scale * (1.44269504088896341f / kK), e);   // what a product is multiplied with
#pragma unroll
        for (int i = 0; i < QW; i++) {
            hf2 hi[4], lo[4];
#pragma unroll
            for (int r = 0; r < 4; r++) split2(ldexpf(x[i][r >> 1][2 * (r & 1)], -e), ldexpf(x[i][r >> 1][2 * (r & 1) + 1], -e), hi[r], lo[r]);
            const hf8 qh = join8(hi[0], hi[1], hi[2], hi[3]), ql = join8(lo[0], lo[1], lo[2], lo[3]);
            if (!mine) continue;
            if constexpr (ST) qs[w * QW + i][0][l] = li < 8 ? qh : ql;
            else qs[w * QW + i][0][l] = qh, qs[w * QW + i][NP - 1][l] = ql;
        }
        lds_barrier();
    }
    hf8 q[NQ][NP];
#pragma unroll
    for (int i = 0; i < NQ; i++)
#pragma unroll
        for (int p = 0; p < NP; p++) q[i][p] = qs[i][p][l];
    f32x4 o[NV];
#pragma unroll
    for (int d = 0; d < NV; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float M = -INFINITY, L = 0.f;
    auto step = [&](int i, u32x4 (&kr)[NS], u32x4 (&vr)[NV], float &s1) {
        const int kt = tile(i), j0 = kt * 64, par = i & 1;
        const bool more = A > 1 || i + A < i1;
        {   // scores
            f32x4 x[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int st = 0; st < NQ; st++) {
                const hf8 k = to_half<E4>(kr[st >> 1][2 * (st & 1)], kr[st >> 1][2 * (st & 1) + 1]);
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) x[st & 1] = mfma16(k, q[st][p], x[st & 1]);
            }
            if (w < 2) {
                sc[par][w][l] = s1 * (w ? kP / 2 : kK);
                if (w) sc[par][2][l] = log2f(fmaxf(s1, 0x1p-99f));
            }
            f32x4 v = x[0] + x[1];
            if constexpr (ST) v = f32x4{add_ror8(v.x), add_ror8(v.y), add_ror8(v.z), add_ror8(v.w)};
            sb[w][l] = v * qsc;
        }
        if (more) load_k(ahead(i), kr, s1);
        lds_barrier();
        {   // weights: the maximum over all keys, the terms of the wavefront's 16
            f32x4 s[4];   // of the sets of 16 keys from w on, around
            float mt = -INFINITY;
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int u = (w + v) & 3;
                s[v] = sb[u][l] * *(const f32x4 *)&sc[par][0][16 * u + 4 * kq];
            }
            if (tile_edge(a, j0, p0, p1))
#pragma unroll
                for (int v = 0; v < 4; v++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int j = j0 + 16 * ((w + v) & 3) + 4 * kq + r;
                        const bool see = j <= pos && (!a.window || j > pos - a.window || j < a.sinks);
                        s[v][r] = see ? s[v][r] : -INFINITY;
                    }
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const f32x4 lv = *(const f32x4 *)&sc[par][2][16 * ((w + v) & 3) + 4 * kq];
#pragma unroll
                for (int r = 0; r < 4; r++) mt = fmaxf(mt, plus(s[v][r], lv[r]));
            }
            mt = max_x16(max_x32(mt));
            float al = 1.f;
            if (mt > M + kGrow || (M == -INFINITY && mt > M)) {   // (the wavefronts agree)
                const float mn = fmaxf(M, mt), h = __builtin_amdgcn_exp2f(0.5f * (M - mn));
                al = h * h;   // (where that is no float any more the total, in steps, still is)
                M = mn;
                L = L * h * h;
            }
            if (w == 0 && kq == 0) alb[li] = al;
            const float ref = M == -INFINITY ? 0.f : M - 1.f;   // (a row that has seen nothing yet: every term is 0)
            const f32x4 vs = *(const f32x4 *)&sc[par][1][16 * w + 4 * kq];
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float p = exp2_twice(fmaf(s[0][r], 0.5f, -0.5f * ref));
                L += p;
                y[r] = p * vs[r];
            }
            hf2 h0, h1, l0, l1;
            split2(y[0], y[1], h0, l0);
            split2(y[2], y[3], h1, l1);
            const hf4 hi = {h0.x, h0.y, h1.x, h1.y}, lo = {l0.x, l0.y, l1.x, l1.y};
            const int at = l * 16 + 8 * (w & 1);
            if constexpr (ST) {   // both column halves hold the row's weights: one keeps each plane
                *(hf4 *)(pb[w >> 1][0] + at) = li < 8 ? hi : lo;
            } else {
                *(hf4 *)(pb[w >> 1][0] + at) = hi;
                *(hf4 *)(pb[w >> 1][NP - 1] + at) = lo;
            }
        }
        lds_barrier();
        // sums
        const float al = alb[li];
        if (__any(al != 1.f))
#pragma unroll
            for (int d = 0; d < NV; d++) o[d] *= al;
        if (E4 && tile_part(j0, a.sinks, lo, last)) {
            const u32x4 m = held_bytes(j0, a.sinks, lo, last);
#pragma unroll
            for (int d = 0; d < NV; d++) vr[d] &= m;
        }
#pragma unroll
        for (int y = 0; y < 2; y++) {
            hf8 p[NP];
#pragma unroll
            for (int x = 0; x < NP; x++) p[x] = *(const hf8 *)(pb[y][x] + l * 16);
#pragma unroll
            for (int d = 0; d < NV; d++) {
                const hf8 v = to_half<E4>(vr[d][2 * y], vr[d][2 * y + 1]);
#pragma unroll
                for (int x = NP - 1; x >= 0; x--) o[d] = mfma16(v, p[x], o[d]);
            }
        }
        if (more) load_v(ahead(i), vr);
    };
    for (int i = i0; i < i1; i += A) {
        step(i, kr[0], vr[0], s1[0]);
        if (A > 1 && i + 1 < i1) step(i + 1, kr[A - 1], vr[A - 1], s1[A - 1]);
    }
    // the rows' totals
    L += __shfl_xor(L, 16, 64);
    L += __shfl_xor(L, 32, 64);
    if (l < 16) mx[w][l] = L;
    lds_barrier();
    if constexpr (ST)
#pragma unroll
        for (int d = 0; d < NV; d++) o[d] = f32x4{add_ror8(o[d].x), add_ror8(o[d].y), add_ror8(o[d].z), add_ror8(o[d].w)};
    if (row >= rows || li >= R) return;
    const float total = (mx[0][li] + mx[1][li]) + (mx[2][li] + mx[3][li]);
    finish<NV>(a, g, row, sp, 16 * w * NV + 4 * kq, M, total, o);   // register r of o[d]: dim 16 (w NV + d) + 4 kq + r
}

// Attention of more rows: 32 by four wavefronts, in a pipeline of three tiles with one barrier a tile: while tile i's scores
// are formed, the weights of tile i - 1 and the sums of tile i - 2 are, all of it independent.
//   scores, weights  16 rows (w >> 1) by 32 keys (w & 1): the rows' queries and the scores stay in registers, the two
//                    wavefronts of the rows exchange their maxima and all of them the weights through LDS
//   sums             a quarter of the dims for all rows
// int8 keys are matrix operands as they are: the queries are integers per row in signed digits of 8 bits (x = X 2^e, |X| <= 2^30),
// every product and sum is exact until the digits' sums are joined in fp32. Three digits hold an element of 2^-k of its row's
// largest to 22 - k bits: at most 2^-19 of the mean magnitude where the largest is 8 times that, as little as fp32's own roundings
// of a score. Work-groups with a row whose largest is above that (a channel far above the others; three digits are off by 1e-4 in a
// weight at 1000 times) take four digits, 30 - k bits, for 3 to 7% of the time.
// 2048 tokens of an empty cache, 16 heads on 4 of 256 dims: 90 to 96 us, 380 TFLOP/s (twice that in matrix instructions' f16 rate); at
// 6144 positions 466 us, 515 (with four digits 97 and 487). Bound by a wavefront's own chain: of a step's 3480 cycles at D = 256 the scores
// take 780, the weights 570, the softmax's end 800, the sums 950 and barrier and loads 350 (before scores and terms took a product more
// each, some 60 cycles), and two work-groups a CU overlap only part of it (the products alone would be 1800 cycles of a SIMD for both, the
// vector instructions 1600). Measured the same or slower: operands of 64 rows shared through LDS, two groups of wavefronts in
// opposite steps, wavefronts with different roles, and the vector instructions placed among the products.
typedef int i32x4 __attribute__((ext_vector_type(4)));
// Four values times 2^(16 - e) as integers, the bytes of X + 0x80808080; each less 128 is one of X's signed digits. Digit p of the four.
__device__ __forceinline__ u32x4 digits(const f32x4 x, int e) {
    u32x4 X;
#pragma unroll
    for (int r = 0; r < 4; r++) X[r] = ((uint32_t)(int)rintf(ldexpf(x[r], 16 - e)) + 0x80808080u) ^ 0x80808080u;
    return X;
}
__device__ __forceinline__ uint32_t digit(const u32x4 X, int p) {
    const uint32_t sel = (uint32_t)p | (uint32_t)(4 + p) << 8 | 0x0c0c0000u;
    return __builtin_amdgcn_perm(X[1], X[0], sel) | __builtin_amdgcn_perm(X[3], X[2], sel) << 16;
}
template <int D, bool E4>
__global__ __launch_bounds__(256, 2) void kv8_chunk_kernel(const Kv8AttnArgs a) {
    constexpr int NS = D / 64, NQ = E4 ? 2 * NS : NS, NP = E4 ? 2 : 3;
    constexpr int CT = 2, NV = D / 64;   // columns; a wavefront's units of values
    __shared__ __align__(16) uint8_t pb[2][CT][2][2][1024];   // weights [tile parity][columns][32 keys][plane][lane]
    __shared__ __align__(16) float sc[4][4][64];             // [tile & 3] scales of the keys times kK, of the values times kP / 2, their log2 (and unused)
    __shared__ float alb[2][CT][16], mx[2][CT][2][16], ms[CT][16];
    __shared__ __align__(16) u32x4 qd[CT][E4 ? 1 : NS][64];   // int8: the queries' fourth digits
    __shared__ int large[4];                                  // int8: a row has a large channel
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, li = l & 15, kq = l >> 4;
    const int cw = w >> 1, u0 = 2 * (w & 1);
    const int G = a.H / a.c.Hkv, rows = a.T * G, np = clamp_past(a.npast, a.npast_dev);
    const int g = blockIdx.x % a.c.Hkv, sp = blockIdx.y, r0 = ((int)gridDim.x / a.c.Hkv - 1 - (int)blockIdx.x / a.c.Hkv) * 32;
    const int p0 = np + r0 / G, p1 = np + min(r0 + 31, rows - 1) / G, last = np + a.T - 1;
    const int lo = a.window ? max(p0 - a.window + 1, 0) : 0;
    const Tiles tl = tiles_of(p0, p1, a.window, a.sinks);
    const int i0 = sp * a.per_split, nt = min(a.per_split, tl.n - i0);
    if (nt <= 0) return;
    const uint8_t *kc = a.c.k + (int64_t)g * a.c.n_tiles * 64 * D + u0 * NS * 1024, *vc = a.c.v + (int64_t)g * a.c.n_tiles * 64 * D + w * NV * 1024;
    const float *scp = (w & 1 ? a.c.vs : a.c.ks) + (((int64_t)g * a.c.n_tiles * 64) >> a.c.lg);
    u32x4 kr[2 * NS], vr[NV];
    float s1;   // even wavefronts: the keys' scale of a tile's position l; odd: the values'
    auto tile = [&](int i) { return i0 + i < tl.ns ? i0 + i : tl.f + i0 + i - tl.ns; };
    auto load_k = [&](int i) { load_units<2 * NS>(kc + (int64_t)tile(min(i, nt - 1)) * 64 * D, l * 16, kr); };
    auto load_v = [&](int i) { load_units<NV>(vc + (int64_t)tile(min(i, nt - 1)) * 64 * D, l * 16, vr); };
    auto load_s = [&](int i) { s1 = scp[min(tile(min(i, nt - 1)) * 64 + l, last) >> a.c.lg]; };
    auto put_s = [&](int i) {   // (every pair of wavefronts the same)
        const float x = held(tile(min(i, nt - 1)) * 64 + l, a.sinks, lo, last) ? s1 : 0.f;
        sc[i & 3][w & 1][l] = x * (w & 1 ? kP / 2 : kK);
        sc[i & 3][2 + (~w & 1)][l] = log2f(fmaxf(x, 0x1p-99f));
    };
    load_s(0);
    load_k(0);
    load_v(0);
    __builtin_amdgcn_sched_barrier(0);
    // the wavefront's queries as operands, an exponent per row; the two wavefronts of the rows prepare them both
    const int rq = min(r0 + 16 * cw + li, rows - 1), tq = rq / G, pos = np + tq;
    u32x4 q[NQ][NP];   // int8: the first three digits
    float qsc;
    {
        const float *qp = a.q + tq * a.q_tok + (g * G + rq % G) * a.q_head + 16 * kq;
        f32x4 x[4 * NS];
        float m = 0.f, sum = 0.f;
        bool fin = true;
#pragma unroll
        for (int i = 0; i < 4 * NS; i++) {
            x[i] = *(const f32x4_u *)(qp + 64 * (i >> 2) + 4 * (i & 3));
#pragma unroll
            for (int r = 0; r < 4; r++) m = fmaxf(m, fabsf(x[i][r])), sum += fabsf(x[i][r]), fin &= fabsf(x[i][r]) < INFINITY;
        }
        m = max_x16(max_x32(m));
        if constexpr (!E4) {
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            large[w] = __any(m * (D / 8) > sum || m < 0x1p-102f);   // (below, where the exponent stops, the bits are needed too)
        }
        const uint64_t bad = ~__ballot(fin);   // a NaN or infinity, which integers do not hold, is put into the row's factor
        fin = !((bad >> li | bad >> (li + 16) | bad >> (li + 32) | bad >> (li + 48)) & 1);
        int e = 0;
        if (m < INFINITY) (void)frexpf(m, &e);   // m < 2^e
        e = max(e, -102) - 14;
        qsc = fin ? ldexpf(a.scale * (1.44269504088896341f / kK), e) : NAN;   // what a product (of int8, its 2^-16) is multiplied with
#pragma unroll
        for (int s = 0; s < NS; s++) {
            if constexpr (E4) {
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    hf2 hi[4], lo[4];
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        split2(ldexpf(x[4 * s + 2 * y + (r >> 1)][2 * (r & 1)], -e), ldexpf(x[4 * s + 2 * y + (r >> 1)][2 * (r & 1) + 1], -e), hi[r], lo[r]);
                    const hf8 qh = join8(hi[0], hi[1], hi[2], hi[3]), ql = join8(lo[0], lo[1], lo[2], lo[3]);
                    __builtin_memcpy(&q[2 * s + y][0], &qh, 16);
                    __builtin_memcpy(&q[2 * s + y][1], &ql, 16);
                }
            } else {
                u32x4 q4;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const u32x4 X = digits(x[4 * s + y], e);
#pragma unroll
                    for (int p = 0; p < 3; p++) q[s][p][y] = digit(X, 3 - p);
                    q4[y] = digit(X, 0);
                }
                if (u0 == 0) qd[cw][s][l] = q4;
            }
        }
    }
    f32x4 o[CT][NV], s[2];   // sums; products of the tile before with its keys' scales
    float M, L, mt;
    put_s(0);
    load_s(1);
    lds_barrier();

    auto tiles = [&](auto n_digits) __attribute__((always_inline)) {
        constexpr int ND = decltype(n_digits)::value;
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int d = 0; d < NV; d++) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        M = mt = -INFINITY, L = 0.f;
        u32x4 q4[ND > 3 ? NS : 1];
        if constexpr (ND > 3)
#pragma unroll
            for (int st = 0; st < NS; st++) q4[st] = qd[cw][st][l];

        // steps of the pipeline: the scores of tile i (S), the weights of tile i - 1 (W), the sums of tile i - 2 (P)
        for (int i = 0; i < nt + 2; i++) {
            const bool S = i < nt, W = i >= 1 && i <= nt, P = i >= 2;
            const int par = i & 1, pw = par ^ 1;   // tile i and i - 2; tile i - 1
            hf8 pf[2][CT];   // weights of half y >> 1, plane 1 - (y & 1): two groups of columns ahead
            auto get_p = [&](int y) {
#pragma unroll
                for (int c = 0; c < CT; c++) pf[y & 1][c] = *(const hf8 *)(pb[par][c][y >> 1][1 - (y & 1)] + l * 16);
            };
            if (P) {
                float al[CT];
#pragma unroll
                for (int c = 0; c < CT; c++) al[c] = alb[par][c][li];
                get_p(0);
                get_p(1);
                bool any = false;
#pragma unroll
                for (int c = 0; c < CT; c++) any |= al[c] != 1.f;
                if (__any(any))
#pragma unroll
                    for (int c = 0; c < CT; c++)
#pragma unroll
                        for (int d = 0; d < NV; d++) o[c][d] *= al[c];
                if (E4) {
                    const int j0 = tile(i - 2) * 64;
                    if (tile_part(j0, a.sinks, lo, last)) {
                        const u32x4 m = held_bytes(j0, a.sinks, lo, last);
#pragma unroll
                        for (int d = 0; d < NV; d++) vr[d] &= m;
                    }
                }
            }
            f32x4 y[2];
            if (S) {
                if constexpr (E4) {
                    f32x4 x[2][2];
#pragma unroll
                    for (int u = 0; u < 2; u++) x[u][0] = x[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int st = 0; st < NQ; st++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const u32x4 &k4 = kr[u * NS + (st >> 1)];
                            const hf8 k = to_half<E4>(k4[2 * (st & 1)], k4[2 * (st & 1) + 1]);
#pragma unroll
                            for (int p = 0; p < 2; p++) {
                                hf8 qq;
                                __builtin_memcpy(&qq, &q[st][p], 16);
                                x[u][p] = mfma16(k, qq, x[u][p]);
                            }
                        }
#pragma unroll
                    for (int u = 0; u < 2; u++) y[u] = x[u][0] + x[u][1];
                } else {
                    i32x4 x[2][ND];
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int p = 0; p < ND; p++) x[u][p] = i32x4{0, 0, 0, 0};
#pragma unroll
                    for (int st = 0; st < NS; st++)
#pragma unroll
                        for (int p = 0; p < ND; p++)
#pragma unroll
                            for (int u = 0; u < 2; u++)
                                x[u][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8((i32x4)kr[u * NS + st], (i32x4)(p < 3 ? q[st][p] : q4[st]), x[u][p], 0, 0, 0);
#pragma unroll
                    for (int u = 0; u < 2; u++)   // a digit's sum is 2^22 at most
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int hi = (x[u][0][r] << 8) + x[u][1][r], lo = ND > 3 ? (x[u][2][r] << 8) + x[u][ND - 1][r] : x[u][2][r];
                            y[u][r] = fmaf((float)lo, ND > 3 ? 0x1p-16f : 0x1p-8f, (float)hi);
                        }
                }
                load_k(i + 1);
            }
            if (W) {
                const float mm = fmaxf(mt, mx[pw][cw][1 - (w & 1)][li]);
                // (the two wavefronts of the rows agree)
                const float mn = mm > M + kGrow || M == -INFINITY ? fmaxf(M, mm) : M;
                const float h = mn == M ? 1.f : __builtin_amdgcn_exp2f(0.5f * (M - mn));
                M = mn;
                L = L * h * h;   // (in steps: a float where h * h may be none)
                alb[pw][cw][li] = h * h;
                const float ref = M == -INFINITY ? 0.f : M - 1.f;   // (a row that has seen nothing yet: every term is 0)
                hf2 hi[4], lo[4];
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const f32x4 vs = *(const f32x4 *)&sc[(i - 1) & 3][1][16 * (u0 + v) + 4 * kq];
                    float z[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float p = exp2_twice(fmaf(s[v][r], 0.5f, -0.5f * ref));
                        L += p;
                        z[r] = p * vs[r];
                    }
                    split2(z[0], z[1], hi[2 * v], lo[2 * v]);
                    split2(z[2], z[3], hi[2 * v + 1], lo[2 * v + 1]);
                }
                *(hf8 *)(pb[pw][cw][w & 1][0] + l * 16) = join8(hi[0], hi[1], hi[2], hi[3]);
                *(hf8 *)(pb[pw][cw][w & 1][1] + l * 16) = join8(lo[0], lo[1], lo[2], lo[3]);
            }
            if (S) {
#pragma unroll
                for (int u = 0; u < 2; u++) s[u] = y[u] * qsc * *(const f32x4 *)&sc[i & 3][0][16 * (u0 + u) + 4 * kq];
                const int j0 = tile(i) * 64;
                if (tile_edge(a, j0, p0, p1))
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int j = j0 + 16 * (u0 + u) + 4 * kq + r;
                            const bool see = j <= pos && (!a.window || j > pos - a.window || j < a.sinks);
                            s[u][r] = see ? s[u][r] : -INFINITY;
                        }
                mt = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const f32x4 lv = *(const f32x4 *)&sc[i & 3][2][16 * (u0 + u) + 4 * kq];
#pragma unroll
                    for (int r = 0; r < 4; r++) mt = fmaxf(mt, plus(s[u][r], lv[r]));
                }
                mt = max_x16(max_x32(mt));
                mx[par][cw][w & 1][li] = mt;
                put_s(i + 1);
                load_s(i + 2);
            }
            if (P) {
                hf8 v[NV];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    if (!(x & 1))
#pragma unroll
                        for (int d = 0; d < NV; d++) v[d] = to_half<E4>(vr[d][x], vr[d][x + 1]);
#pragma unroll
                    for (int d = 0; d < NV; d++)
#pragma unroll
                        for (int c = 0; c < CT; c++) o[c][d] = mfma16(v[d], pf[x & 1][c], o[c][d]);
                    if (x < 2) get_p(x + 2);
                }
                load_v(i - 1);
            }
            lds_barrier();
        }
    };
    int four = E4 ? 0 : __builtin_amdgcn_readfirstlane(large[0] | large[2]);
    if (!four) tiles(std::integral_constant<int, 3>{});
    if (!E4) asm volatile("" : "+s"(four));   // (as one choice of two the loops take 20 registers more, and spill at D = 256)
    if (four) tiles(std::integral_constant<int, 4>{});
    // the rows' totals
    L += __shfl_xor(L, 16, 64);
    L += __shfl_xor(L, 32, 64);
    if (l < 16) {
        mx[0][cw][w & 1][l] = L;
        if (u0 == 0) ms[cw][l] = M;
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int row = r0 + 16 * c + li;   // register r of o[d]: dim 16 (w NV + d) + 4 kq + r
        if (row < rows) finish<NV>(a, g, row, sp, 16 * w * NV + 4 * kq, ms[c][li], mx[0][c][0][li] + mx[0][c][1][li], o[c]);
    }
}

// The splits of a row joined in order: W wavefronts take every W-th split each (a lane D / 64 dims), their sums are added in
// order. W = 1: four rows per work-group. Latency bound: 63 splits of 16 rows of 256 3.9 us, 128 5.3; a launch alone is 3.
template <int D, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void kv8_merge_kernel(const Kv8AttnArgs a, int R) {
    constexpr int V = D / 64;
    typedef float vec __attribute__((ext_vector_type(V)));
    __shared__ float red[W][V][64], rl[W];
    const int tid = threadIdx.x, l = tid & 63, w = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.H / a.c.Hkv, rows = a.T * G, rr = W == 1 ? (int)blockIdx.x * 4 + (tid >> 6) : (int)blockIdx.x, g = blockIdx.y;
    if (rr >= rows) return;
    const int np = clamp_past(a.npast, a.npast_dev), r0 = rr / R * R;
    const Tiles tl = tiles_of(np + r0 / G, np + min(r0 + R - 1, rows - 1) / G, a.window, a.sinks);
    const int ns = (tl.n + a.per_split - 1) / a.per_split;
    const float *part = a.part + ((int64_t)g * rows + rr) * a.n_split * (D + 4);
    const int t = rr / G, h = g * G + rr % G;
    constexpr int U = 8;
    vec v[U];
    float m[U], c[U];
    auto load = [&](int s) {   // (past the end: the last one again, with weight 0)
#pragma unroll
        for (int i = 0; i < U; i++) {
            const float *p = part + (int64_t)min(s + i * W, ns - 1) * (D + 4);
            m[i] = p[0];
            c[i] = p[1];
            __builtin_memcpy(&v[i], p + 4 + V * l, sizeof(vec));
        }
    };
    vec gate = 0.f;
    float M = -INFINITY;
    if (l < ns) M = part[(int64_t)l * (D + 4)];
    load(w);   // with the maxima
    if (a.gate && w == 0) __builtin_memcpy(&gate, a.gate + t * a.g_tok + h * a.g_head + V * l, sizeof(vec));
    for (int s = l + 64; s < ns; s += 64) M = fmaxf(M, part[(int64_t)s * (D + 4)]);
    M = xjd::wave_max(M);
    vec y = 0.f;
    float L = 0.f;
    for (int s = w; s < ns; s += U * W) {
        if (s > w) load(s);
#pragma unroll
        for (int i = 0; i < U; i++) {
            const float h = s + i * W >= ns || m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(0.5f * (m[i] - M)), f = h * h;   // (as the kernels rescale)
            L = fmaf(h * c[i], h, L);
            if (f > 0.f) y += v[i] * f;
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int i = 0; i < V; i++) red[w][i][l] = V == 1 ? ((float *)&y)[0] : ((float *)&y)[i];
        if (l == 0) rl[w] = L;
        __syncthreads();
        if (w) return;
        L = 0.f;
        y = 0.f;
#pragma unroll
        for (int x = 0; x < W; x++) {
            L += rl[x];
#pragma unroll
            for (int i = 0; i < V; i++) ((float *)&y)[i] += red[x][i][l];
        }
    }
    y *= (2.f / kP) / L;
    float *op = a.out + t * a.o_tok + (int64_t)h * D + V * l;
    if (a.gate)
#pragma unroll
        for (int i = 0; i < V; i++) ((float *)&y)[i] *= sigm_fast(((float *)&gate)[i]);
#pragma unroll
    for (int i = 0; i < V; i++) op[i] = ((float *)&y)[i];
}

// Tiles that R rows see at most.
static int most_tiles(const Kv8AttnArgs &a, int R) {
    const int all = (a.npast + a.T - 1) / 64 + 1;
    if (!a.window) return all;
    const int G = a.H / a.c.Hkv, span = (R + G - 1) / G + 1;   // tokens of R rows
    const int64_t n = ((int64_t)a.sinks + 63) / 64 + ((int64_t)a.window + span + 62) / 64 + 1;
    return n < all ? (int)n : all;
}
// Rows of a work-group (times of 16 heads on 4 of 256 dims, int8, as replayed graphs). Up to 8 share every product between their planes,
// half the matrix instructions: one token of 32 heads on as many of 128 dims at 32000 positions 65 us, 69 as 16 rows. 16 is the
// kernel that shares a tile's work out, the shorter way through it, 32 the one that has more rows in a pass over the cache: up to 16 rows
// the first (4 tokens at 131000: 58 us, 61 as 32), and as long as its work-groups have a tile each (5 tokens at 200 positions 9.4 us,
// 12.3 as 32; 64 at 0 7.0 and 9.9; 16 at 1000, 256 of them, 12.2 and 14.1; beyond: 32 at 4000, 2016, 20.6 and 19.8, 64 at 8000 43 and
// 35; not measured between). With e4m3 the scores of 32 rows are no integer products, and 16 rows hold out for 20 D tiles (of 256
// dims 64 tokens at 4000 25.5 and 26.5, of 128 at 2000, 2112 tiles, 15.1 and 15.2, 128 at 2000, 4352 tiles, 21.3 and 20.8, of 64 on 8
// heads 40 at 4000, 1536 tiles, 13.0 and 12.1).
static int64_t groups16(const Kv8AttnArgs &a) { return ((int64_t)a.T * (a.H / a.c.Hkv) + 15) / 16 * a.c.Hkv; }
static int rows_of(const Kv8AttnArgs &a) {
    const int64_t n = (int64_t)a.T * (a.H / a.c.Hkv);
    return n <= 8 ? 8 : n <= 16 || groups16(a) * most_tiles(a, 16) <= (a.c.e4m3 ? 20 * a.c.D : 512) ? 16 : 32;
}
// Splits of the tiles (times in us of 16 heads on 4 of 256 dims, int8, as replayed graphs).
//   Up to three tiles: none, the merge costs more than it saves (one token at 64 positions 8.5 split and 7.6 not, at 128 8.7 and
//   8.9, at 192 8.6 and 10.3; 32 as 32 rows at 128 12.9 and 12.5).
//   Two work-groups a CU, which their registers leave room for, hide each other's waits: 512 in all.
//   Up to 16 rows a tile each is enough (for 256, 384, 512 and 768 work-groups one token at 131000 takes 70, 60, 56 and 57, four 77, 66,
//   58 and 67). The merge reads every split: 256 at most (16 heads on one, one token at 32000 in 128, 256 and 512 16.5, 16.8 and
//   22), and above 64 half as many, once, where they would have less than two and a half tiles each: with four kv heads 64 for 128
//   (one token at 5000, 79 tiles, in 40 splits 10.3 and in 79 11.8, at 12000 in 63 13.5 and in 94 15.1, at 24000 in 63 18.3 and in
//   126 17.5), with one or two 128 for 256, where 64 would be the better on one side only (8 heads on 2, one token at 5000 in
//   79 splits 10.6 and in 40 10.1, at 12000 in 94 12.5 and in 63 11.6, but at 4200 in 66 9.9 and in 33 10.5, at 16000 in 126 12.9 and in
//   63 13.8). Of 64 dims, whose registers leave room for more, 1024 up to 128
//   splits (32 heads on 8 at 131000 43 with 512 and 36 with 1024; 16 on 4 at 32000 13.1 in 128 splits and 15.2 in 256).
//   More rows, up to 128 groups of them: 512 if each has four tiles (for 256 and 512: 8 tokens at 131000 78 and 68, 200 at 2000 35 and
//   32), else 256 of two at least (at three tiles in 512 or in between 40 at 4000 22 and 25; a number in between leaves
//   some CUs one work-group and others two).
//   From 129 groups on the other choice is no split and no merge (256 dims; of fewer the last paragraph decides first where a group
//   has enough tiles): worth five tiles a third up to 170 (333 tokens at 500 29.0 whole, 29.6 in thirds, at 1000 40.0 and 34.5), twelve
//   a half or a third beyond (512 at 500 33.5 whole, 37.1 in halves, at 2000 64 and 59, at 32000 684 and 515; 600, thirds in two
//   turns, at 1000 48 and 54, at 2000 77 and 73, at 32000 912 and 636).
//   Of 128 and 64 dims a CU holds three and four of these, which take eight tiles each and at most 64 splits (128 dims, for 512 and 768 in
//   all: 512 tokens at 32000 351 and 320, 128 at 4000, five tiles, 25.7 and 26.6, 8 at 131000, 64 and 96 splits, 44.1 and
//   45.7; 64 dims, 32 heads on 8, for 512 and 1024: 256 at 32000 313 and 248).
static int64_t splits_few(const Kv8AttnArgs &a, int64_t wgs, int tiles) {
    int64_t n = 512 / wgs;
    if (a.c.D == 64) n = std::max(n, std::min<int64_t>(1024 / wgs, 128));
    n = std::min<int64_t>(n, 256);
    if (n > 64 && 2 * tiles < 5 * n) n = std::max<int64_t>(n / 2, 64);
    return std::min<int64_t>(n, tiles);
}
static int splits_of(const Kv8AttnArgs &a) {
    const int R = rows_of(a), tiles = most_tiles(a, R);
    const int64_t rows = (int64_t)a.T * (a.H / a.c.Hkv), wgs = (rows + R - 1) / R * a.c.Hkv;
    if (tiles <= 3) return 1;
    if (R < 32) return std::max<int64_t>(splits_few(a, wgs, tiles), 1);
    for (int per = a.c.D == 64 ? 4 : a.c.D == 128 ? 3 : 2; per > 1; per--) {
        const int64_t n = (per == 2 && wgs > 256 && wgs <= 341 ? 1024 : 256 * per) / wgs;
        if (tiles >= (wgs > 170 ? 12 : per > 2 ? 8 : wgs > 128 ? 5 : 4) * n && (per == 2 || n <= 64)) return n < 1 ? 1 : (int)n;
    }
    return (int)std::max<int64_t>(std::min<int64_t>(256 / wgs, (tiles + 1) / 2), 1);
}
int64_t kv8_attn_part_floats(const Kv8AttnArgs &a) {
    int64_t n = splits_of(a);
    if (most_tiles(a, 16) > 3) n = std::max(n, splits_few(a, groups16(a), most_tiles(a, 16)));   // what fewer tiles may take as 16 rows
    return n > 1 ? (int64_t)a.T * a.H * n * (a.c.D + 4) : 0;
}

template <int D, bool E4>
static void attn_launch_d(const Kv8AttnArgs &a, int R, hipStream_t st) {
    const int rows = a.T * (a.H / a.c.Hkv);
    const dim3 grid((rows + R - 1) / R * a.c.Hkv, a.n_split);
    // Two tiles ahead where a tile is small and a work-group has some: one token of 32 heads on as many of 128 dims at 32000 positions, 32
    // tiles, 57 us with two and 68 with one, at 8000, 8 tiles, 19.4 and 20.4; of 16 heads on 4 at 32000, 4 tiles, 15.4 and 15.2, at 4000,
    // one tile, 8.7 and 8.5; of 256 dims, whose registers then leave a CU fewer work-groups, on 4 heads at 131000 60 and 58.
    constexpr int A = D < 256 ? 2 : 1;
    const bool ahead = A > 1 && a.per_split >= 6;
    if (R == 8 && ahead) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 8, A>), grid, dim3(256), 0, st, a);
    else if (R == 8) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 8, 1>), grid, dim3(256), 0, st, a);
    else if (R == 16 && ahead) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 16, A>), grid, dim3(256), 0, st, a);
    else if (R == 16) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 16, 1>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_chunk_kernel<D, E4>), grid, dim3(256), 0, st, a);
    if (a.n_split == 1) return;
    // eight wavefronts a row where there is more than a round of one's loads and the rows do not fill the GPU by themselves (one token at
    // 576 positions, 10 splits, 9.8 us with one and 9.4 with eight, at 256, 5 splits, 8.6 and 9.1; 64 of 8 heads of 64 dims at 500 9.3 and 10.2)
    if (a.n_split <= 8 || rows * a.c.Hkv > (a.n_split <= 16 ? 256 : 1024)) hipLaunchKernelGGL((kv8_merge_kernel<D, 1>), dim3((rows + 3) / 4, a.c.Hkv), dim3(256), 0, st, a, R);
    else hipLaunchKernelGGL((kv8_merge_kernel<D, 8>), dim3(rows, a.c.Hkv), dim3(512), 0, st, a, R);
}

int kv8_attn_launch(const Kv8AttnArgs &in, int64_t part_floats, hipStream_t st) {
    Kv8AttnArgs a = in;
    int64_t n = splits_of(a), cap = part_floats / ((int64_t)a.T * a.H * (a.c.D + 4));
    if (n > cap) n = cap;
    if (n < 1) n = 1;
    const int R = rows_of(a), tiles = most_tiles(a, R);
    a.per_split = (int)((tiles + n - 1) / n);
    a.n_split = (tiles + a.per_split - 1) / a.per_split;
    switch (a.c.D) {
    case 64: a.c.e4m3 ? attn_launch_d<64, true>(a, R, st) : attn_launch_d<64, false>(a, R, st); break;
    case 128: a.c.e4m3 ? attn_launch_d<128, true>(a, R, st) : attn_launch_d<128, false>(a, R, st); break;
    case 256: a.c.e4m3 ? attn_launch_d<256, true>(a, R, st) : attn_launch_d<256, false>(a, R, st); break;
    default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int D>
static void store_launch_d(const Kv8StoreArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.T + 62) >> 6) + 1, a.c.Hkv, 2);   // tiles of T rows from any position
    if (a.c.e4m3) hipLaunchKernelGGL((kv8_store_kernel<D, true>), grid, dim3(2 * D), 0, st, a);
    else hipLaunchKernelGGL((kv8_store_kernel<D, false>), grid, dim3(2 * D), 0, st, a);
}
int kv8_store_launch(const Kv8StoreArgs &a, hipStream_t st) {
    switch (a.c.D) {
    case 64: store_launch_d<64>(a, st); break;
    case 128: store_launch_d<128>(a, st); break;
    case 256: store_launch_d<256>(a, st); break;
    default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// Two groups a thread (16 bytes of a dim's values) where the work-groups take turns on the CUs: 32000 positions of 4 heads of 256
// 65 us, 69 with one; one where all are there at once: 77 positions of one head of 128 3.1 us, 3.9 with two, 2100 of 4 of 256 6.0 and 7.0.
template <int D, bool E4>
static void load_launch_d(const Kv8LoadArgs &a, hipStream_t st) {
    const dim3 grid(((a.pos0 + a.n - 1) >> 6) - (a.pos0 >> 6) + 1, a.c.Hkv, a.k && a.v ? 2 : 1);
    if ((int64_t)grid.x * grid.y * grid.z > 1024) hipLaunchKernelGGL((kv8_load_kernel<D, E4, 2>), grid, dim3(D), 0, st, a);
    else hipLaunchKernelGGL((kv8_load_kernel<D, E4, 1>), grid, dim3(2 * D), 0, st, a);
}
int kv8_load_launch(const Kv8LoadArgs &a, hipStream_t st) {
    switch (a.c.D) {
    case 64: a.c.e4m3 ? load_launch_d<64, true>(a, st) : load_launch_d<64, false>(a, st); break;
    case 128: a.c.e4m3 ? load_launch_d<128, true>(a, st) : load_launch_d<128, false>(a, st); break;
    case 256: a.c.e4m3 ? load_launch_d<256, true>(a, st) : load_launch_d<256, false>(a, st); break;
    default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace xjk
