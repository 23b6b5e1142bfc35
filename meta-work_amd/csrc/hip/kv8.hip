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

namespace xjk {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
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
// The code of x: nearest to the exact quotient x / s, ties to even.
//   int8: rint of the product with 1 / s is at most one off; the rest x - c s
//   is exact in one fma (it is below s and a multiple of the smaller ulp), so comparing
//   it with s / 2 decides.
//   e4m3: s is a power of two, the product with 1 / s is exact and converts to nearest even.
template <bool E4>
__device__ __forceinline__ uint32_t code_of(float x, float s, float inv) {
    if constexpr (E4) {
        float y = x * inv;
        y = fminf(fmaxf(y, -448.f), 448.f);
        if (x != x || s == 0.f) y = 0.f;
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xFFu;
    } else {
        if (x != x || s == 0.f) return 0;
        float c = rintf(fminf(fmaxf(x * inv, -127.f), 127.f));
        const float r2 = 2.f * fmaf(-c, s, x);
        if (r2 > s || (r2 == s && ((int)c & 1))) c += 1.f;
        else if (r2 < -s || (r2 == -s && ((int)c & 1))) c -= 1.f;
        c = fminf(fmaxf(c, -127.f), 127.f);
        return (uint32_t)(int)c & 0xFFu;
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

// Store and load move a tile in groups of 16 positions by D / 4 lanes, a lane 4 dims, so that the float rows
// (four times the codes' bytes) go 16 bytes per lane and whole rows per instruction. Group q of the
// keys is the 16 positions of one unit row; of the values the positions 16 u + 4 q + r, whose codes of a dim
// are 16 bytes.
template <bool VAL>
__device__ __forceinline__ int group_pos(int q, int i) { return VAL ? 16 * (i >> 2) + 4 * q + (i & 3) : 16 * q + i; }

// The lane's codes: w[i] byte c = dim d0 + c of the group's position i.
template <int D, bool VAL>
__device__ __forceinline__ void get_codes(const uint8_t *tile, int q, int d0, uint32_t (&w)[16]) {
    if constexpr (VAL) {
        const uint8_t *p = tile + (d0 >> 4) * 1024 + q * 256 + (d0 & 15) * 16;
        u32x4 v[4];
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = *(const u32x4 *)(p + 16 * c);
#pragma unroll
        for (int u = 0; u < 4; u++) {   // 4 dims x 4 positions turned
            const uint32_t a = __builtin_amdgcn_perm(v[1][u], v[0][u], 0x05010400u), b = __builtin_amdgcn_perm(v[1][u], v[0][u], 0x07030602u);
            const uint32_t c = __builtin_amdgcn_perm(v[3][u], v[2][u], 0x05010400u), d = __builtin_amdgcn_perm(v[3][u], v[2][u], 0x07030602u);
            w[4 * u] = __builtin_amdgcn_perm(c, a, 0x05040100u);
            w[4 * u + 1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
            w[4 * u + 2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
            w[4 * u + 3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
        }
    } else {
        const uint8_t *p = tile + q * (16 * D) + (d0 >> 6) * 1024 + ((d0 >> 4) & 3) * 256 + (d0 & 15);
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = *(const uint32_t *)(p + 16 * i);
    }
}
template <int D, bool VAL>
__device__ __forceinline__ void put_codes(uint8_t *tile, int q, int d0, const uint32_t (&w)[16]) {
    if constexpr (VAL) {
        uint8_t *p = tile + (d0 >> 4) * 1024 + q * 256 + (d0 & 15) * 16;
        u32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const uint32_t a = __builtin_amdgcn_perm(w[4 * u + 1], w[4 * u], 0x05010400u), b = __builtin_amdgcn_perm(w[4 * u + 1], w[4 * u], 0x07030602u);
            const uint32_t c = __builtin_amdgcn_perm(w[4 * u + 3], w[4 * u + 2], 0x05010400u), d = __builtin_amdgcn_perm(w[4 * u + 3], w[4 * u + 2], 0x07030602u);
            v[0][u] = __builtin_amdgcn_perm(c, a, 0x05040100u);
            v[1][u] = __builtin_amdgcn_perm(c, a, 0x07060302u);
            v[2][u] = __builtin_amdgcn_perm(d, b, 0x05040100u);
            v[3][u] = __builtin_amdgcn_perm(d, b, 0x07060302u);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) *(u32x4 *)(p + 16 * c) = v[c];
    } else {
        uint8_t *p = tile + q * (16 * D) + (d0 >> 6) * 1024 + ((d0 >> 4) & 3) * 256 + (d0 & 15);
#pragma unroll
        for (int i = 0; i < 16; i++) *(uint32_t *)(p + 16 * i) = w[i];
    }
}
// The largest of D / 4 consecutive lanes, in each of them.
template <int D>
__device__ __forceinline__ float row_max(float v) {
    v = xjd::row16_max(v);
    if (D >= 128) v = fmaxf(v, __shfl_xor(v, 16, 64));
    if (D >= 256) v = fmaxf(v, __shfl_xor(v, 32, 64));
    return v;
}

// A work-group stores one tile of a kv head's keys or values (D threads, a group each D / 4): the
// rows' largest magnitudes, joined over every block in LDS, the scales, the codes. In a
// tile that is not new from end to end the codes of the other positions are read
// and written back as they are, those of a begun block at its new scale if that grew.
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
    uint32_t w[16];
    if (!whole) get_codes<D, VAL>(tile, q, d0, w);
    f32x4 y[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int p = j0 + group_pos<VAL>(q, i);
        y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p >= np && p < end) y[i] = *(const f32x4_u *)(x + (int64_t)(p - np) * tok);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float m = row_max<D>(fmaxf(fmaxf(finite_abs(y[i].x), finite_abs(y[i].y)), fmaxf(finite_abs(y[i].z), finite_abs(y[i].w))));
        if (d0 == 0) sm[0][group_pos<VAL>(q, i)] = m;
    }
    __syncthreads();
    if (tid < 64) {   // position j0 + tid: sm[0] its block's scale, sm[1] the block's earlier scale if it is begun
        float m = sm[0][tid];
        for (int o = 1; o < B; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const int first = (j0 + tid) & -B;
        float s = block_scale<E4>(m), old = 0.f;
        if (first < np && first + B > np) {
            old = sp[tid >> a.c.lg];
            s = fmaxf(s, old);
        }
        sm[0][tid] = s;
        sm[1][tid] = old;
        if ((tid & (B - 1)) == 0 && first < end && first + B > np) sp[tid >> a.c.lg] = s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int pl = group_pos<VAL>(q, i), p = j0 + pl;
        const float s = sm[0][pl], inv = s > 0.f ? 1.f / s : 0.f;
        if (whole || (p >= np && p < end)) {
            w[i] = code_of<E4>(y[i].x, s, inv) | code_of<E4>(y[i].y, s, inv) << 8 | code_of<E4>(y[i].z, s, inv) << 16 | code_of<E4>(y[i].w, s, inv) << 24;
        } else if (p < np && (p | (B - 1)) >= np) {
            const float old = sm[1][pl];
            if (s > old)
                w[i] = recode<E4>(w[i] & 0xFFu, old, s) | recode<E4>(w[i] >> 8 & 0xFFu, old, s) << 8 |
                       recode<E4>(w[i] >> 16 & 0xFFu, old, s) << 16 | recode<E4>(w[i] >> 24, old, s) << 24;
        }
    }
    put_codes<D, VAL>(tile, q, d0, w);
}
template <int D, bool E4>
__global__ __launch_bounds__(D) void kv8_store_kernel(const Kv8StoreArgs a) {
    __shared__ float sm[2][64];
    if (blockIdx.z) store_tile<D, E4, true>(a, sm);
    else store_tile<D, E4, false>(a, sm);
}

template <int D, bool E4, bool VAL>
__device__ __forceinline__ void load_tile(const Kv8LoadArgs &a) {
    const int g = blockIdx.y, tid = threadIdx.x, q = tid / (D / 4), d0 = tid % (D / 4) * 4;
    const int kt = (a.pos0 >> 6) + blockIdx.x, j0 = kt * 64;
    const float *sp = (VAL ? a.c.vs : a.c.ks) + ((((int64_t)g * a.c.n_tiles + kt) * 64) >> a.c.lg);
    uint32_t w[16];
    get_codes<D, VAL>((VAL ? a.c.v : a.c.k) + ((int64_t)g * a.c.n_tiles + kt) * 64 * D, q, d0, w);
    float *y = (VAL ? a.v : a.k) + g * D + d0;
    const int64_t tok = VAL ? a.v_tok : a.k_tok;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int pl = group_pos<VAL>(q, i), t = j0 + pl - a.pos0;
        if (t < 0 || t >= a.n) continue;
        const float s = sp[pl >> a.c.lg];
        *(f32x4_u *)(y + t * tok) = f32x4{value_of<E4>(w[i] & 0xFFu, s), value_of<E4>(w[i] >> 8 & 0xFFu, s), value_of<E4>(w[i] >> 16 & 0xFFu, s),
                                          value_of<E4>(w[i] >> 24, s)};
    }
}
template <int D, bool E4>
__global__ __launch_bounds__(D) void kv8_load_kernel(const Kv8LoadArgs a) {
    if (a.k && !(a.v && blockIdx.z)) load_tile<D, E4, false>(a);
    else load_tile<D, E4, true>(a);
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
    lo = __builtin_convertvector(f32x2{y0 - (float)hi.x, y1 - (float)hi.y}, hf2);   // the differences are exact
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
// enters as two f16 planes of w * kP (22 bits), whatever the scales' range, the total is of
// 2^(score - M). The sums are rescaled only when max t passes M by more than kGrow.
constexpr float kGrow = 8.f, kP = 128.f;

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
// The lane's bytes of a values unit at j0 that positions after `last` do not hold: an e4m3 code not written yet may be a NaN,
// which a weight of 0 does not take out.
__device__ __forceinline__ u32x4 written(int j0, int last) {
    const int kq = (threadIdx.x & 63) >> 4;
    u32x4 m;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int n = last + 1 - (j0 + 16 * u + 4 * kq);
        m[u] = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
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

// N groups of 4 sums, 16 dims apart from dim d0 of the token's head: over the total, gated, into the output row at hd.
template <int N>
__device__ __forceinline__ void finish_row(const Kv8AttnArgs &a, int t, int h, int64_t hd, int d0, float total, const f32x4 *o) {
    const float inv = (1.f / kP) / total;
    float *op = a.out + t * a.o_tok + hd + d0;
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

// Attention: a work-group takes R query rows (row = token * G + head of the kv head) and a split of the tiles. Its four
// wavefronts share every tile, each a part of every step, so nothing is converted or summed twice:
//   scores   16 keys each, for all rows: K units from the cache to registers, the queries stay in registers
//   weights  a quarter of the (row, key) pairs each: scores and weights pass through LDS (a few KB a tile)
//   sums     a quarter of the dims each, for all rows
// A wavefront's part of the next tile (8 KB at D = 256) is always in flight. Two to four work-groups share a CU: one's
// vector instructions (conversions, softmax) run beside another's products, which they outweigh (D = 256, R = 32: 260
// against 64 products of 16 cycles a tile).
// An operand has 16 columns. R = 8: both planes of 8 rows, so a product costs one instruction; more: 16 rows, the planes one
// after the other, R / 16 sets of columns.
template <int D, bool E4, int R>
__global__ __launch_bounds__(256, 2) void kv8_attn_kernel(const Kv8AttnArgs a) {
    constexpr int NS = D / 64, NV = D / 64, NQ = 2 * NS;   // a wavefront's units of keys and of values; 32-dim steps of a score
    constexpr bool ST = R == 8;
    constexpr int CT = ST ? 1 : R / 16, NP = ST ? 1 : 2;   // sets of columns, operands per set
    constexpr int QW = NQ >= 4 ? NQ / 4 : 1;               // steps whose queries a wavefront prepares
    __shared__ __align__(16) hf8 qs[CT][NQ][NP][64];
    __shared__ __align__(16) f32x4 sb[CT][4][64];          // scores [columns][16 keys][lane]
    __shared__ __align__(16) uint8_t pb[CT][2][NP][1024];  // weights as operands [columns][32 keys][plane][lane]
    __shared__ __align__(16) float sc[2][3][64];           // [tile parity] scales of the keys, of the values times kP, their log2
    __shared__ float alb[CT][16], mx[CT][4][16], ms[CT][16];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, li = l & 15, kq = l >> 4;
    const int G = a.H / a.c.Hkv, rows = a.T * G, np = clamp_past(a.npast, a.npast_dev);
    // the rows with the most tiles first
    const int g = blockIdx.x % a.c.Hkv, sp = blockIdx.y, r0 = ((int)gridDim.x / a.c.Hkv - 1 - (int)blockIdx.x / a.c.Hkv) * R;
    const int p0 = np + r0 / G, p1 = np + min(r0 + R - 1, rows - 1) / G, last = np + a.T - 1;
    const Tiles tl = tiles_of(p0, p1, a.window, a.sinks);
    const int i0 = sp * a.per_split, i1 = min(i0 + a.per_split, tl.n);
    if (i0 >= tl.n) return;
    const uint8_t *kc = a.c.k + (int64_t)g * a.c.n_tiles * 64 * D + w * NS * 1024, *vc = a.c.v + (int64_t)g * a.c.n_tiles * 64 * D + w * NV * 1024;
    const int64_t s0 = ((int64_t)g * a.c.n_tiles * 64) >> a.c.lg;
    u32x4 kr[NS], vr[NV];
    float s1 = 0.f;   // wavefront 0: the keys' scale of position l; 1: the values'
    auto tile = [&](int i) { return i < tl.ns ? i : tl.f + i - tl.ns; };
    auto load_k = [&](int kt) {   // positions not written yet have no scale
        load_units<NS>(kc + (int64_t)kt * 64 * D, l * 16, kr);
        const int j = kt * 64 + l;
        if (w < 2) s1 = j <= last ? (w ? a.c.vs : a.c.ks)[s0 + (j >> a.c.lg)] : 0.f;
    };
    auto load_v = [&](int kt) { load_units<NV>(vc + (int64_t)kt * 64 * D, l * 16, vr); };
    load_k(tile(i0));
    load_v(tile(i0));
    __builtin_amdgcn_sched_barrier(0);
    auto query = [&](int c, int &t, int &h) {   // the lane's row in a set of columns
        const int rr = min(r0 + 16 * c + (li & (R - 1)), rows - 1);
        t = rr / G;
        h = g * G + rr % G;
    };
    // the queries as operands, step i = 2 s + e the dims 64 s + 16 kq + 8 e .. + 7, x 2^-e = hi + lo, e per row
    {
        f32x4 x[CT][QW][2];
        const bool mine = w * QW < NQ;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            int t, h;
            query(c, t, h);
            const float *q = a.q + t * a.q_tok + h * a.q_head + 16 * kq;
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < QW; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int st = mine ? w * QW + i : 0;
                    x[c][i][e] = *(const f32x4_u *)(q + 64 * (st >> 1) + 8 * (st & 1) + 4 * e);
#pragma unroll
                    for (int r = 0; r < 4; r++) m = fmaxf(m, fabsf(x[c][i][e][r]));
                }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if (l < 16) mx[c][w][l] = m;
        }
        lds_barrier();
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const float m = fmaxf(fmaxf(mx[c][0][li], mx[c][1][li]), fmaxf(mx[c][2][li], mx[c][3][li]));
            int e = 0;
            if (m < INFINITY) (void)frexpf(m, &e);   // m < 2^e
            e = max(e, -100) - 14;
            if (l < 16 && w == 0) ms[c][l] = ldexpf(a.scale * 1.44269504088896341f, e);   // what a product is multiplied with
#pragma unroll
            for (int i = 0; i < QW; i++) {
                hf2 hi[4], lo[4];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    split2(ldexpf(x[c][i][r >> 1][2 * (r & 1)], -e), ldexpf(x[c][i][r >> 1][2 * (r & 1) + 1], -e), hi[r], lo[r]);
                const hf8 qh = join8(hi[0], hi[1], hi[2], hi[3]), ql = join8(lo[0], lo[1], lo[2], lo[3]);
                if (!mine) continue;
                if constexpr (ST) qs[c][w * QW + i][0][l] = li < 8 ? qh : ql;
                else qs[c][w * QW + i][0][l] = qh, qs[c][w * QW + i][NP - 1][l] = ql;
            }
        }
        lds_barrier();
    }
    hf8 q[CT][NQ][NP];
    f32x4 o[CT][NV];
#pragma unroll
    for (int c = 0; c < CT; c++) {
#pragma unroll
        for (int i = 0; i < NQ; i++)
#pragma unroll
            for (int p = 0; p < NP; p++) q[c][i][p] = qs[c][i][p][l];
#pragma unroll
        for (int d = 0; d < NV; d++) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // the wavefront's part of the weights: CT of the four sets of 16 keys, from u0, of the columns cw
    const int cw = (w * CT) >> 2, u0 = (w * CT) & 3;
    const float qsc = ms[cw][li];
    int tw, hw;
    query(cw, tw, hw);
    const int pos = np + tw;
    float M = -INFINITY, L = 0.f;
    for (int i = i0; i < i1; i++) {
        const int kt = tile(i), j0 = kt * 64, par = i & 1;
        const bool more = i + 1 < i1;
        {   // scores
            f32x4 x[CT];
#pragma unroll
            for (int c = 0; c < CT; c++) x[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NQ; st++) {
                const hf8 k = to_half<E4>(kr[st >> 1][2 * (st & 1)], kr[st >> 1][2 * (st & 1) + 1]);
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                    for (int c = 0; c < CT; c++) x[c] = mfma16(k, q[c][st][p], x[c]);
            }
            if (w < 2) {
                sc[par][w][l] = w ? s1 * kP : s1;
                if (w) sc[par][2][l] = log2f(fmaxf(s1, 0x1p-100f));
            }
#pragma unroll
            for (int c = 0; c < CT; c++) {
                f32x4 v = x[c];
                if constexpr (ST) v = f32x4{add_ror8(v.x), add_ror8(v.y), add_ror8(v.z), add_ror8(v.w)};
                sb[c][w][l] = v;
            }
        }
        if (more) load_k(tile(i + 1));
        lds_barrier();
        {   // weights
            f32x4 s[4];
            float mt = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const f32x4 ks = *(const f32x4 *)&sc[par][0][16 * u + 4 * kq];
                s[u] = sb[cw][u][l];
#pragma unroll
                for (int r = 0; r < 4; r++) s[u][r] *= qsc * ks[r];
            }
            if (tile_edge(a, j0, p0, p1))
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int j = j0 + 16 * u + 4 * kq + r;
                        if (j > pos || (a.window && j <= pos - a.window && j >= a.sinks)) s[u][r] = -INFINITY;
                    }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const f32x4 lv = *(const f32x4 *)&sc[par][2][16 * u + 4 * kq];
#pragma unroll
                for (int r = 0; r < 4; r++) mt = fmaxf(mt, s[u][r] + lv[r]);
            }
            mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
            float al = 1.f;
            if (mt > M + kGrow || (M == -INFINITY && mt > M)) {   // (the wavefronts of the same columns agree)
                const float mn = fmaxf(M, mt);
                al = __builtin_amdgcn_exp2f(M - mn);
                M = mn;
                L *= al;
            }
            if (u0 == 0 && kq == 0) alb[cw][li] = al;
            const float ref = M == -INFINITY ? 0.f : M;   // (a row that has seen nothing yet: every term is 0)
#pragma unroll
            for (int v = 0; v < CT; v++) {
                const int u = u0 + v;
                f32x4 x = s[v];
                if (CT < 4)   // s[u0 + v] without a register index that varies
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if (y == u) x = s[y];
                const f32x4 vs = *(const f32x4 *)&sc[par][1][16 * u + 4 * kq];
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float p = __builtin_amdgcn_exp2f(x[r] - ref);
                    L += p;
                    y[r] = p * vs[r];
                }
                hf2 h0, h1, l0, l1;
                split2(y[0], y[1], h0, l0);
                split2(y[2], y[3], h1, l1);
                typedef _Float16 hf4 __attribute__((ext_vector_type(4)));
                const hf4 hi = {h0.x, h0.y, h1.x, h1.y}, lo = {l0.x, l0.y, l1.x, l1.y};
                const int at = l * 16 + 8 * (u & 1);
                if constexpr (ST) {
                    *(hf4 *)(pb[cw][u >> 1][0] + at) = li < 8 ? hi : lo;
                } else {
                    *(hf4 *)(pb[cw][u >> 1][0] + at) = hi;
                    *(hf4 *)(pb[cw][u >> 1][NP - 1] + at) = lo;
                }
            }
        }
        lds_barrier();
        {   // sums
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const float al = alb[c][li];
                if (__any(al != 1.f))
#pragma unroll
                    for (int d = 0; d < NV; d++) o[c][d] *= al;
            }
            if (E4 && j0 + 63 > last) {
                const u32x4 m = written(j0, last);
#pragma unroll
                for (int d = 0; d < NV; d++) vr[d] &= m;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                hf8 p[CT][NP];
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int x = 0; x < NP; x++) p[c][x] = *(const hf8 *)(pb[c][h][x] + l * 16);
#pragma unroll
                for (int d = 0; d < NV; d++) {
                    const hf8 v = to_half<E4>(vr[d][2 * h], vr[d][2 * h + 1]);
#pragma unroll
                    for (int x = NP - 1; x >= 0; x--)
#pragma unroll
                        for (int c = 0; c < CT; c++) o[c][d] = mfma16(v, p[c][x], o[c][d]);
                }
            }
            if (more) load_v(tile(i + 1));
        }
    }
    // the rows' totals
    L += __shfl_xor(L, 16, 64);
    L += __shfl_xor(L, 32, 64);
    if (l < 16) {
        mx[cw][CT == 4 ? 0 : w % (4 / CT)][l] = L;
        if (u0 == 0) ms[cw][l] = M;
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < CT; c++) {
        if constexpr (ST)
#pragma unroll
            for (int d = 0; d < NV; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[c][d][r] = add_ror8(o[c][d][r]);
        const int row = r0 + 16 * c + li;
        if (row >= rows || li >= R) continue;
        float total = mx[c][0][li];
#pragma unroll
        for (int x = 1; x < 4 / CT; x++) total += mx[c][x][li];
        const int d0 = 16 * w * NV + 4 * kq;   // register r of o[d]: dim 16 (w NV + d) + 4 kq + r
        if (a.n_split > 1) {
            float *part = a.part + (((int64_t)g * rows + row) * a.n_split + sp) * (D + 4);
            if (w == 0 && kq == 0) part[0] = ms[c][li], part[1] = total;
#pragma unroll
            for (int d = 0; d < NV; d++) *(f32x4 *)(part + 4 + d0 + 16 * d) = o[c][d];
        } else {
            const int h = g * G + row % G;
            finish_row<NV>(a, row / G, h, h * D, d0, total, o[c]);
        }
    }
}

// The splits of a row joined in order: W wavefronts take every W-th split each (a lane D / 64 dims), their sums are added in
// order. W = 1: four rows per work-group.
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
    float M = -INFINITY;
    for (int s = l; s < ns; s += 64) M = fmaxf(M, part[(int64_t)s * (D + 4)]);
    M = xjd::wave_max(M);
    vec y = 0.f;
    float L = 0.f;
    constexpr int U = 8;
    for (int s = w; s < ns; s += U * W) {
        vec v[U];
        float m[U], c[U];
#pragma unroll
        for (int i = 0; i < U; i++) {   // (past the end: the last one again, with weight 0)
            const float *p = part + (int64_t)min(s + i * W, ns - 1) * (D + 4);
            m[i] = p[0];
            c[i] = p[1];
            __builtin_memcpy(&v[i], p + 4 + V * l, sizeof(vec));
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            const float f = s + i * W >= ns || m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - M);
            L = fmaf(f, c[i], L);
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
    y *= (1.f / kP) / L;
    float *op = a.out + t * a.o_tok + (int64_t)h * D + V * l;
    if (a.gate) {
        const float *gp = a.gate + t * a.g_tok + h * a.g_head + V * l;
#pragma unroll
        for (int i = 0; i < V; i++) ((float *)&y)[i] *= sigm_fast(gp[i]);
    }
#pragma unroll
    for (int i = 0; i < V; i++) op[i] = ((float *)&y)[i];
}

// Rows of a work-group: up to 8 rows share every product between their planes (half the matrix instructions); as many as
// there are, up to what the queries' registers allow (32 of 256 dims, 64 of fewer).
static int rows_of(const Kv8AttnArgs &a) {
    const int64_t n = (int64_t)a.T * (a.H / a.c.Hkv);
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 || a.c.D == 256 ? 32 : 64;
}
// Tiles that R rows see at most.
static int most_tiles(const Kv8AttnArgs &a, int R) {
    const int all = (a.npast + a.T - 1) / 64 + 1;
    if (!a.window) return all;
    const int G = a.H / a.c.Hkv, span = (R + G - 1) / G + 1;   // tokens of R rows
    const int64_t n = ((int64_t)a.sinks + 63) / 64 + ((int64_t)a.window + span + 62) / 64 + 1;
    return n < all ? (int)n : all;
}
// Splits of the tiles while the work-groups do not exceed what the CUs hold.
static int splits_of(const Kv8AttnArgs &a) {
    const int R = rows_of(a), tiles = most_tiles(a, R);
    const int64_t rows = (int64_t)a.T * (a.H / a.c.Hkv), wgs = (rows + R - 1) / R * a.c.Hkv;
    int64_t n = (R >= 32 ? 512 : 768) / wgs;
    if (n > tiles) n = tiles;
    return n < 1 ? 1 : (int)n;
}
int64_t kv8_attn_part_floats(const Kv8AttnArgs &a) {
    const int n = splits_of(a);
    return n > 1 ? (int64_t)a.T * a.H * n * (a.c.D + 4) : 0;
}

template <int D, bool E4>
static void attn_launch_d(const Kv8AttnArgs &a, int R, hipStream_t st) {
    const int rows = a.T * (a.H / a.c.Hkv), nb = (rows + R - 1) / R;
    const dim3 grid(nb * a.c.Hkv, a.n_split);
    if (R == 8) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 8>), grid, dim3(256), 0, st, a);
    else if (R == 16) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 16>), grid, dim3(256), 0, st, a);
    else if (R == 32) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 32>), grid, dim3(256), 0, st, a);
    else if constexpr (D < 256) hipLaunchKernelGGL((kv8_attn_kernel<D, E4, 64>), grid, dim3(256), 0, st, a);
    if (a.n_split == 1) return;
    if (a.n_split <= 16 || rows * a.c.Hkv > 1024) hipLaunchKernelGGL((kv8_merge_kernel<D, 1>), dim3((rows + 3) / 4, a.c.Hkv), dim3(256), 0, st, a, R);
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
    if (a.c.e4m3) hipLaunchKernelGGL((kv8_store_kernel<D, true>), grid, dim3(D), 0, st, a);
    else hipLaunchKernelGGL((kv8_store_kernel<D, false>), grid, dim3(D), 0, st, a);
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

template <int D>
static void load_launch_d(const Kv8LoadArgs &a, hipStream_t st) {
    const dim3 grid(((a.pos0 + a.n - 1) >> 6) - (a.pos0 >> 6) + 1, a.c.Hkv, a.k && a.v ? 2 : 1);
    if (a.c.e4m3) hipLaunchKernelGGL((kv8_load_kernel<D, true>), grid, dim3(D), 0, st, a);
    else hipLaunchKernelGGL((kv8_load_kernel<D, false>), grid, dim3(D), 0, st, a);
}
int kv8_load_launch(const Kv8LoadArgs &a, hipStream_t st) {
    switch (a.c.D) {
    case 64: load_launch_d<64>(a, st); break;
    case 128: load_launch_d<128>(a, st); break;
    case 256: load_launch_d<256>(a, st); break;
    default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace xjk
