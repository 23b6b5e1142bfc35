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
// 16 codes as two operands of 8.
template <bool E4>
__device__ __forceinline__ void to_half(u32x4 w, hf8 &a, hf8 &b) {
    hf2 h[8];
#pragma unroll
    for (int i = 0; i < 4; i++) to_half4<E4>(w[i], h[2 * i], h[2 * i + 1]);
    a = join8(h[0], h[1], h[2], h[3]);
    b = join8(h[4], h[5], h[6], h[7]);
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

// A lane's part of its query row as operands, step (s, e) the dims 64 s + 16 kq + 8 e .. + 7, x 2^-e = hi + lo. Returns what
// a product of them is multiplied with: the row's 2^e, the scale and log2 e.
template <int D>
__device__ __forceinline__ float split_query(const float *q, float scale, hf8 (&qh)[D / 32], hf8 (&ql)[D / 32]) {
    f32x4 x[D / 16];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; i++) x[i] = *(const f32x4_u *)(q + 64 * (i >> 2) + 4 * (i & 3));
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) m = fmaxf(m, fabsf(x[i][c]));
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    int e = 0;
    if (m < INFINITY) (void)frexpf(m, &e);   // m < 2^e
    e = max(e, -100) - 14;
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
        hf2 hi[4], lo[4];
#pragma unroll
        for (int c = 0; c < 4; c++)
            split2(ldexpf(x[2 * i + (c >> 1)][2 * (c & 1)], -e), ldexpf(x[2 * i + (c >> 1)][2 * (c & 1) + 1], -e), hi[c], lo[c]);
        qh[i] = join8(hi[0], hi[1], hi[2], hi[3]);
        ql[i] = join8(lo[0], lo[1], lo[2], lo[3]);
    }
    return ldexpf(scale * 1.44269504088896341f, e);
}

// The softmax of a tile's scores: s (products so far) becomes the weights' planes. sc: the tile's scales (keys, values times
// kP, log2 of the values'); edge: some row does not see the whole tile.
template <int ND>
__device__ __forceinline__ void tile_weights(const Kv8AttnArgs &a, f32x4 (&s)[4], const float (*sc)[64], float qsc, int j0, int pos, bool edge,
                                             float &M, float &L, f32x4 (&o)[ND], hf8 (&ph)[2], hf8 (&pl)[2]) {
    const int kq = (threadIdx.x & 63) >> 4;
    float mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const f32x4 ks = *(const f32x4 *)&sc[0][16 * u + 4 * kq];
#pragma unroll
        for (int r = 0; r < 4; r++) s[u][r] *= qsc * ks[r];
    }
    if (edge)
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int j = j0 + 16 * u + 4 * kq + r;
                if (j > pos || (a.window && j <= pos - a.window && j >= a.sinks)) s[u][r] = -INFINITY;
            }
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const f32x4 lv = *(const f32x4 *)&sc[2][16 * u + 4 * kq];
#pragma unroll
        for (int r = 0; r < 4; r++) mt = fmaxf(mt, s[u][r] + lv[r]);
    }
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    if (__any(mt > M + kGrow || (M == -INFINITY && mt > M))) {
        const float mn = fmaxf(M, mt), al = mn == M ? 1.f : __builtin_amdgcn_exp2f(M - mn);
        M = mn;
        L *= al;
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] *= al;
    }
    const float ms = M == -INFINITY ? 0.f : M;   // (a row that has seen nothing yet: every term is 0)
    hf2 hi[8], lo[8];
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const f32x4 vs = *(const f32x4 *)&sc[1][16 * u + 4 * kq];
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float p = __builtin_amdgcn_exp2f(s[u][r] - ms);
            L += p;
            y[r] = p * vs[r];
        }
        split2(y[0], y[1], hi[2 * u], lo[2 * u]);
        split2(y[2], y[3], hi[2 * u + 1], lo[2 * u + 1]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        ph[i] = join8(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
        pl[i] = join8(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
    }
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

// Attention of few rows (row = token * G + head of the kv head): a work-group takes R of them and a split of the tiles. Its
// four wavefronts share every tile: each forms the scores of 16 keys, all of them (through LDS) the weights of
// all 64, each the sums of a quarter of the dims, so that a short context's one tile takes a quarter of the time and a wavefront
// needs few registers (four on a SIMD hide the loads). Every wavefront always has its part of the next
// tile in flight, 8 KB at D = 256. With R = 8 an operand's 16 columns are both planes of the 8 rows, so a product costs
// one instruction; with R = 16 the planes follow one another, with R = 32 there are two sets of columns.
template <int D, bool E4, int R>
__global__ __launch_bounds__(256, R == 32 ? 2 : 3) void kv8_rows_kernel(const Kv8AttnArgs a) {
    constexpr int NS = D / 64, NV = D / 64, CT = R == 32 ? 2 : 1;   // a wavefront's units of keys and of values; column sets
    constexpr bool ST = R == 8;
    __shared__ __align__(16) float sc[2][3][64];
    __shared__ __align__(16) f32x4 sb[2][CT][4][64];   // [tile parity][columns][16 keys][lane]
    __shared__ __align__(16) hf8 qs[ST ? 1 : CT][ST ? 1 : 2 * NS][2][64];   // the queries' planes, if not in registers
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, li = l & 15, kq = l >> 4;
    const int g = blockIdx.y, sp = blockIdx.z, G = a.H / a.c.Hkv, rows = a.T * G;
    const int np = clamp_past(a.npast, a.npast_dev);
    const int r0 = blockIdx.x * R, t0 = r0 / G, t1 = min(r0 + R - 1, rows - 1) / G;
    const Tiles tl = tiles_of(np + t0, np + t1, a.window, a.sinks);
    const int i0 = sp * a.per_split, i1 = min(i0 + a.per_split, tl.n);
    if (i0 >= tl.n) return;
    const int last = np + a.T - 1;
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
    hf8 q8[2 * NS];   // R = 8: the lane's plane
    float qsc[CT], M[CT], L[CT];
    int row[CT], pos[CT];
    f32x4 o[CT][NV];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        row[c] = r0 + 16 * c + (li & (R - 1));
        const int rr = min(row[c], rows - 1), t = rr / G, h = g * G + rr % G;
        pos[c] = np + t;
        hf8 qh[2 * NS], ql[2 * NS];
        qsc[c] = split_query<D>(a.q + t * a.q_tok + h * a.q_head + 16 * kq, a.scale, qh, ql);
#pragma unroll
        for (int i = 0; i < 2 * NS; i++) {
            if constexpr (ST) q8[i] = li < 8 ? qh[i] : ql[i];
            else if (i % 4 == w) qs[c][i][0][l] = qh[i], qs[c][i][1][l] = ql[i];
        }
        M[c] = -INFINITY;
        L[c] = 0.f;
#pragma unroll
        for (int d = 0; d < NV; d++) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (!ST) lds_barrier();
    for (int i = i0; i < i1; i++) {
        const int kt = tile(i), j0 = kt * 64, par = i & 1;
        const bool more = i + 1 < i1;
        f32x4 x[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) x[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < NS; st++) {
            hf8 ka, kb;
            to_half<E4>(kr[st], ka, kb);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                if constexpr (ST) {
                    x[c] = mfma16(ka, q8[2 * st], x[c]);
                    x[c] = mfma16(kb, q8[2 * st + 1], x[c]);
                } else {
                    x[c] = mfma16(ka, qs[c][2 * st][1][l], x[c]);
                    x[c] = mfma16(kb, qs[c][2 * st + 1][1][l], x[c]);
                    x[c] = mfma16(ka, qs[c][2 * st][0][l], x[c]);
                    x[c] = mfma16(kb, qs[c][2 * st + 1][0][l], x[c]);
                }
            }
        }
        if (w < 2) {
            sc[par][w][l] = w ? s1 * kP : s1;
            if (w) sc[par][2][l] = log2f(fmaxf(s1, 0x1p-100f));
        }
#pragma unroll
        for (int c = 0; c < CT; c++) {
            if constexpr (ST)
#pragma unroll
                for (int r = 0; r < 4; r++) x[c][r] = add_ror8(x[c][r]);
            sb[par][c][w][l] = x[c];
        }
        if (more) load_k(tile(i + 1));
        lds_barrier();   // (the other parity: one barrier a tile)
        hf8 ph[CT][2], pl[CT][2];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            f32x4 s[4];
#pragma unroll
            for (int u = 0; u < 4; u++) s[u] = sb[par][c][u][l];
            tile_weights(a, s, sc[par], qsc[c], j0, pos[c], tile_edge(a, j0, np + t0, np + t1), M[c], L[c], o[c], ph[c], pl[c]);
            if constexpr (ST) {   // both column halves hold the row's weights: one keeps each plane
                if (li >= 8) ph[c][0] = pl[c][0], ph[c][1] = pl[c][1];
            }
        }
        if (E4 && j0 + 63 > last) {
            const u32x4 m = written(j0, last);
#pragma unroll
            for (int d = 0; d < NV; d++) vr[d] &= m;
        }
#pragma unroll
        for (int d = 0; d < NV; d++) {
            hf8 va, vb;
            to_half<E4>(vr[d], va, vb);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                if constexpr (!ST) {
                    o[c][d] = mfma16(va, pl[c][0], o[c][d]);
                    o[c][d] = mfma16(vb, pl[c][1], o[c][d]);
                }
                o[c][d] = mfma16(va, ph[c][0], o[c][d]);
                o[c][d] = mfma16(vb, ph[c][1], o[c][d]);
            }
        }
        if (more) load_v(tile(i + 1));
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {
        L[c] += __shfl_xor(L[c], 16, 64);
        L[c] += __shfl_xor(L[c], 32, 64);
        if constexpr (ST)
#pragma unroll
            for (int d = 0; d < NV; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[c][d][r] = add_ror8(o[c][d][r]);
        if (row[c] >= rows || li >= R) continue;
        // register r of o[d]: dim 16 (w NV + d) + 4 kq + r
        const int d0 = 16 * w * NV + 4 * kq;
        if (a.n_split > 1) {
            float *part = a.part + (((int64_t)g * rows + row[c]) * a.n_split + sp) * (D + 4);
            if (w == 0 && kq == 0) part[0] = M[c], part[1] = L[c];
#pragma unroll
            for (int d = 0; d < NV; d++) *(f32x4 *)(part + 4 + d0 + 16 * d) = o[c][d];
        } else {
            const int t = row[c] / G, h = g * G + row[c] % G;
            finish_row<NV>(a, t, h, h * D, d0, L[c], o[c]);
        }
    }
}

// Attention of many rows: a work-group takes 64 query rows of a kv head, its two groups of four wavefronts (16 rows each)
// every other tile. A tile's codes become f16 operands in LDS once for the four wavefronts (64 KB at D = 256, in operand
// order: every access is 64 consecutive 16-byte pieces). Per tile a group has a step on the vector units (the softmax of the
// tile's scores; its values and the next tile's keys turned into operands) and one on the matrix cores (its values'
// products, then the next tile's scores); the groups take them in turn, one a step behind the other,
// so that on every SIMD one wavefront keeps the matrix core busy while the other has the vector unit.
template <int D, bool E4>
__global__ __launch_bounds__(512, 2) void kv8_chunk_kernel(const Kv8AttnArgs a) {
    constexpr int NS = D / 64, ND = D / 16, NU = D / 64;   // units of keys (and of values) per wavefront: 4 NS / 4 = ND / 4
    __shared__ __align__(16) uint8_t Ks[2][64 * D * 2], Vs[2][64 * D * 2];
    __shared__ __align__(16) float sc[2][2][3][64];   // [group][tile parity]
    __shared__ float ml[2][2][64];
    const int tid = threadIdx.x, l = tid & 63, li = l & 15, kq = l >> 4;
    const int grp = __builtin_amdgcn_readfirstlane(tid >> 8), w = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
    const int G = a.H / a.c.Hkv, rows = a.T * G, b = blockIdx.x;
    const int g = b % a.c.Hkv, sp = blockIdx.y, r0 = ((int)gridDim.x / a.c.Hkv - 1 - b / a.c.Hkv) * 64;   // the most tiles first
    const int np = clamp_past(a.npast, a.npast_dev), last = np + a.T - 1;
    const Tiles tl = tiles_of(np + r0 / G, np + min(r0 + 63, rows - 1) / G, a.window, a.sinks);
    const int i0 = sp * a.per_split, nt = min(a.per_split, tl.n - i0);
    if (nt <= 0) return;
    const int rw = r0 + 16 * w, row = min(rw + li, rows - 1), t = row / G, h = g * G + row % G, pos = np + t;
    const int p0 = np + min(rw, rows - 1) / G, p1 = np + min(rw + 15, rows - 1) / G;   // the wavefront's rows
    const uint8_t *kc = a.c.k + (int64_t)g * a.c.n_tiles * 64 * D, *vc = a.c.v + (int64_t)g * a.c.n_tiles * 64 * D;
    const int64_t s0 = ((int64_t)g * a.c.n_tiles * 64) >> a.c.lg;
    const int n = (nt + 1 - grp) / 2;   // the group's tiles
    auto tile = [&](int j) {
        const int i = i0 + grp + 2 * j;
        return i < tl.ns ? i : tl.f + i - tl.ns;
    };
    u32x4 kr[NU], vr[NU];
    float k1 = 0.f, v1 = 0.f;
    auto load_k = [&](int j) {
        const int kt = tile(j), p = kt * 64 + l;
        load_units<NU>(kc + (int64_t)kt * 64 * D + w * NU * 1024, l * 16, kr);
        if (w == 0) {
            const bool in = p <= last;
            k1 = in ? a.c.ks[s0 + (p >> a.c.lg)] : 0.f;
            v1 = in ? a.c.vs[s0 + (p >> a.c.lg)] : 0.f;
        }
    };
    if (n > 0) load_k(0);
    hf8 qh[2 * NS], ql[2 * NS];
    const float qsc = split_query<D>(a.q + t * a.q_tok + h * a.q_head + 16 * kq, a.scale, qh, ql);
    f32x4 o[ND], s[4];
    hf8 ph[2], pl[2];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float M = -INFINITY, L = 0.f;
    for (int x = 0; x < nt + 3; x++) {   // 2 n + 2 steps of either group, the second's one later
        const int step = x - grp, j = step >> 1;
        if (step >= 0 && !(step & 1) && j <= n) {
            if (j > 0) {   // tile j - 1: softmax, values
                const int j0 = tile(j - 1) * 64;
                tile_weights(a, s, sc[grp][(j - 1) & 1], qsc, j0, pos, tile_edge(a, j0, p0, p1), M, L, o, ph, pl);
                if (E4 && j0 + 63 > last) {
                    const u32x4 m = written(j0, last);
#pragma unroll
                    for (int c = 0; c < NU; c++) vr[c] &= m;
                }
#pragma unroll
                for (int c = 0; c < NU; c++) {
                    hf8 x, y;
                    to_half<E4>(vr[c], x, y);
                    *(hf8 *)(Vs[grp] + (w * NU + c) * 2048 + l * 16) = x;
                    *(hf8 *)(Vs[grp] + (w * NU + c) * 2048 + 1024 + l * 16) = y;
                }
            }
            if (j < n) {   // the keys of tile j
#pragma unroll
                for (int c = 0; c < NU; c++) {
                    hf8 x, y;
                    to_half<E4>(kr[c], x, y);
                    *(hf8 *)(Ks[grp] + (w * NU + c) * 2048 + l * 16) = x;
                    *(hf8 *)(Ks[grp] + (w * NU + c) * 2048 + 1024 + l * 16) = y;
                }
                if (w == 0) {
                    sc[grp][j & 1][0][l] = k1;
                    sc[grp][j & 1][1][l] = v1 * kP;
                    sc[grp][j & 1][2][l] = log2f(fmaxf(v1, 0x1p-100f));
                }
            }
        }
        if (step >= 0 && (step & 1) && j <= n) {
            if (j < n) load_units<NU>(vc + (int64_t)tile(j) * 64 * D + w * NU * 1024, l * 16, vr);
            if (j + 1 < n) load_k(j + 1);
            if (j > 0)
#pragma unroll
                for (int d = 0; d < ND; d += 2) {
                    hf8 v[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) v[c] = *(const hf8 *)(Vs[grp] + d * 2048 + c * 1024 + l * 16);
                    o[d] = mfma16(v[0], pl[0], o[d]);
                    o[d + 1] = mfma16(v[2], pl[0], o[d + 1]);
                    o[d] = mfma16(v[1], pl[1], o[d]);
                    o[d + 1] = mfma16(v[3], pl[1], o[d + 1]);
                    o[d] = mfma16(v[0], ph[0], o[d]);
                    o[d + 1] = mfma16(v[2], ph[0], o[d + 1]);
                    o[d] = mfma16(v[1], ph[1], o[d]);
                    o[d + 1] = mfma16(v[3], ph[1], o[d + 1]);
                }
            if (j < n) {
#pragma unroll
                for (int u = 0; u < 4; u++) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < 2 * NS; st++) {
                    hf8 ka[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) ka[u] = *(const hf8 *)(Ks[grp] + (u * 2 * NS + st) * 1024 + l * 16);
#pragma unroll
                    for (int u = 0; u < 4; u++) s[u] = mfma16(ka[u], ql[st], s[u]);
#pragma unroll
                    for (int u = 0; u < 4; u++) s[u] = mfma16(ka[u], qh[st], s[u]);
                }
            }
        }
        lds_barrier();
    }
    // the groups' sums joined: each hands the other half of its dims over and finishes the rest
    L += __shfl_xor(L, 16, 64);
    L += __shfl_xor(L, 32, 64);
    if (kq == 0) {
        ml[grp][0][16 * w + li] = M;
        ml[grp][1][16 * w + li] = L;
    }
    lds_barrier();
    const float m2 = ml[grp ^ 1][0][16 * w + li], l2 = ml[grp ^ 1][1][16 * w + li], mm = fmaxf(M, m2);
    const float f1 = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mm), f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mm);
    const float ll = grp ? l2 * f2 + L * f1 : L * f1 + l2 * f2;   // (the same sum in both)
    f32x4 *xo = (f32x4 *)Ks;   // [receiving group][wavefront][ND / 2][64]
#pragma unroll
    for (int d = 0; d < ND; d++) {
        o[d] *= f1;
        if ((d >= ND / 2) != grp) xo[(((grp ^ 1) * 4 + w) * (ND / 2) + d % (ND / 2)) * 64 + l] = o[d];
    }
    lds_barrier();
    if (rw + li >= rows) return;
    float *part = a.part + (((int64_t)g * rows + row) * a.n_split + sp) * (D + 4);
    if (a.n_split > 1 && kq == 0 && grp == 0) part[0] = mm, part[1] = ll;
    auto give = [&](int d1, const f32x4 *half) {   // register r of o[d]: dim 16 d + 4 kq + r
        f32x4 v[ND / 2];
#pragma unroll
        for (int d = 0; d < ND / 2; d++) {
            v[d] = half[d] + xo[((grp * 4 + w) * (ND / 2) + d) * 64 + l];
            if (a.n_split > 1) *(f32x4 *)(part + 4 + 16 * (d1 + d) + 4 * kq) = v[d];
        }
        if (a.n_split == 1) finish_row<ND / 2>(a, t, h, (int64_t)h * D, 16 * d1 + 4 * kq, ll, v);
    };
    if (grp == 0) give(0, o);
    else give(ND / 2, o + ND / 2);
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

// Rows of a work-group: up to 8 rows share every product between their planes (half the matrix instructions), up to 32
// take the kernel without operand tiles in LDS.
static int rows_of(const Kv8AttnArgs &a) {
    const int64_t n = (int64_t)a.T * (a.H / a.c.Hkv);
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64;
}
// Tiles that R rows see at most.
static int most_tiles(const Kv8AttnArgs &a, int R) {
    const int all = (a.npast + a.T - 1) / 64 + 1;
    if (!a.window) return all;
    const int G = a.H / a.c.Hkv, span = (R + G - 1) / G + 1;   // tokens of R rows
    const int64_t n = ((int64_t)a.sinks + 63) / 64 + ((int64_t)a.window + span + 62) / 64 + 1;
    return n < all ? (int)n : all;
}
// Splits of the tiles: work-groups for every CU to hold (64 rows: one, of up to 8 wavefronts; fewer: three or four), and four
// tiles for each of 64 rows, whose partial sums cost as much as a tile.
static int splits_of(const Kv8AttnArgs &a) {
    const int R = rows_of(a);
    const int64_t rows = (int64_t)a.T * (a.H / a.c.Hkv), wgs = (rows + R - 1) / R * a.c.Hkv;
    const int by_tiles = R == 64 ? (most_tiles(a, R) + 3) / 4 : most_tiles(a, R);
    int64_t n = (R == 64 ? 256 : R == 32 ? 512 : 768) / wgs;
    if (n > by_tiles) n = by_tiles;
    return n < 1 ? 1 : (int)n;
}
int64_t kv8_attn_part_floats(const Kv8AttnArgs &a) {
    const int n = splits_of(a);
    return n > 1 ? (int64_t)a.T * a.H * n * (a.c.D + 4) : 0;
}

template <int D, bool E4>
static void attn_launch_d(const Kv8AttnArgs &a, int R, hipStream_t st) {
    const int rows = a.T * (a.H / a.c.Hkv), nb = (rows + R - 1) / R;
    if (R == 8) hipLaunchKernelGGL((kv8_rows_kernel<D, E4, 8>), dim3(nb, a.c.Hkv, a.n_split), dim3(256), 0, st, a);
    else if (R == 16) hipLaunchKernelGGL((kv8_rows_kernel<D, E4, 16>), dim3(nb, a.c.Hkv, a.n_split), dim3(256), 0, st, a);
    else if (R == 32) hipLaunchKernelGGL((kv8_rows_kernel<D, E4, 32>), dim3(nb, a.c.Hkv, a.n_split), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv8_chunk_kernel<D, E4>), dim3(nb * a.c.Hkv, a.n_split), dim3(512), 0, st, a);
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
