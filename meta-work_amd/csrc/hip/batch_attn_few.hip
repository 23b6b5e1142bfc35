// Attention for requests of few rows (gfx950): single tokens and short drafts over pages, short prompts. See batch_attn.h.
#include "batch_attn.h"
#include <algorithm>

namespace xjk {

// A tile of 16 rows, the key tiles of the piece dealt to four wavefronts, which join at the end. Lane l: li = l & 15, kq = l >> 4.
// Keys come straight into the operand's registers (key li, dims 32 s + 8 kq ..); values are read as
// the lane's VW dims of the eight keys whose weights it holds and turned in registers. A tile's keys are requested as soon as the scores of
// the one before are there, its values behind that one's sums. Weights enter in two planes at least (in the kernel for
// many rows those of 16-bit rows in one): the matrix cores wait for memory here. By the trace a token at 131000 positions of 4 heads of 256 in f16, 537 MB,
// takes 96 us (5.6 TB/s), 64 tokens at 1 to 16000 positions of 8 heads of 128 in bf16, 502 MB, 110 us.
template <int D, class E, int NP, int RT, bool PAGES>
__global__ __launch_bounds__(256) void attn_few_kernel(const BatchAttnArgs a) {
    typedef typename Row<RT>::t R;
    constexpr int NS = D / 32, VW = D >= 128 ? 8 : 4, NB = D / (16 * VW), PAD = D + 4, NW = NP > 2 ? NP : 2;
    __shared__ __align__(16) float so[4][16][PAD];
    __shared__ float sm[4][16], sl[4][16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, kq = lane >> 4;
    Item it;
    if (!find_item<kFewRows, kFewKeys, false>(a, blockIdx.x, it)) return;
    const int row = it.tile * 16 + li, n_rows = it.s.rows * a.G, last = min(it.tile * 16 + 15, n_rows - 1);
    const int rq = min(row, n_rows - 1), tok = token_of(a, rq), p = it.s.pos0 + tok;
    const int pf = it.s.pos0 + token_of(a, it.tile * 16), pl = it.s.pos0 + token_of(a, last);
    const Range g = range_of<kFewKeys>(a, pf, pl);
    const int i0 = part_from(g.n, it.piece, it.pieces) + w, i1 = part_from(g.n, it.piece + 1, it.pieces);

    // ---- a tile: its pages, keys and values
    const int32_t *tab = PAGES ? a.table + (int64_t)it.s.r * a.max_blocks : nullptr;
    struct Pages {
        int j0, page[2];
    };
    auto pages_of = [&](int i) {
        Pages x;
        x.j0 = g.tile(min(i, i1 - 1)) * kFewKeys;
#pragma unroll
        for (int u = 0; u < 2; u++) x.page[u] = PAGES ? page_at(a, tab, x.j0 + 16 * u) : 0;
        return x;
    };
    auto at = [&](const Pages &x, int u) {   // of a page that is none, page 0's, which counts for nothing
        const int j = x.j0 + 16 * u;
        return (((((int64_t)max(x.page[u], 0) * a.Hkv + it.head) << a.lg) + (j & ((1 << a.lg) - 1)))) * D;
    };
    V8<E> kf[2][NS];
    uint32_t vv[8][NB][VW / 2];
    auto load_keys = [&](const Pages &x) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if constexpr (PAGES) {
                const E *kp = (const E *)a.k + at(x, u) + li * D + 8 * kq;
#pragma unroll
                for (int s = 0; s < NS; s++) kf[u][s] = *(const V8<E> *)(kp + 32 * s);
            } else {   // behind the last row, the last one, which counts for nothing there
                const E *kp = (const E *)a.k + (it.s.start + min(x.j0 + 16 * u + li, it.s.rows - 1)) * a.k_tok + it.head * a.k_head + 8 * kq;
#pragma unroll
                for (int s = 0; s < NS; s++) kf[u][s] = __builtin_bit_cast(V8<E>, *(const Rows<E, 8> *)(kp + 32 * s));
            }
        }
    };
    auto load_values = [&](const Pages &x) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if constexpr (PAGES) {
                const E *vp = (const E *)a.v + at(x, u) + 4 * kq * D + VW * li;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int b = 0; b < NB; b++) __builtin_memcpy(vv[4 * u + r][b], __builtin_assume_aligned(vp + r * D + 16 * VW * b, 2 * VW), 2 * VW);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const E *vp = (const E *)a.v + (it.s.start + min(x.j0 + 16 * u + 4 * kq + r, it.s.rows - 1)) * a.v_tok + it.head * a.v_head + VW * li;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const Rows<E, VW> y = *(const Rows<E, VW> *)(vp + 16 * VW * b);
                        __builtin_memcpy(vv[4 * u + r][b], &y, 2 * VW);
                    }
                }
            }
        }
    };
    // ---- queries, with the scale's sign; float ones scaled to 2^14 .. 2^15 before they become f16 planes
    Rows<R, 8> x[NS];
    {
        const R *qp = (const R *)a.q + (it.s.start + tok) * a.q_tok + (it.head * a.G + rq - tok * a.G) * a.q_head + 8 * kq;
#pragma unroll
        for (int s = 0; s < NS; s++) x[s] = *(const Rows<R, 8> *)(qp + 32 * s);
    }
    Pages now{}, next{};
    if (i0 < i1) {
        now = pages_of(i0);
        load_keys(now);
        load_values(now);
        next = pages_of(i0 + 4);
    }
    V8<E> q[NS][NP];
    float c = fabsf(a.scale) * 1.44269504088896340736f, up = a.scale < 0.f ? -1.f : 1.f;
    if constexpr (NP == 2) {
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf((float)x[s][i]));
        top = max_x32(max_x16(top));
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
    }
    f32x4 o[D / 16];
#pragma unroll
    for (int d = 0; d < D / 16; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;   // m: a whole number, so that every rescaling is exact
    const float lift = lift_of<E, kFewKeys>(it.s), raised = __builtin_amdgcn_exp2f(lift);

    for (int i = i0; i < i1; i += 4) {
        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; st++)
#pragma unroll
                for (int k = NP - 1; k >= 0; k--) s[u] = Op<E>::mfma16(kf[u][st], q[st][k], s[u]);
        }
        const int j0 = now.j0;
        const bool ok[2] = {now.page[0] >= 0, now.page[1] >= 0};
        now = next;
        if (i + 4 < i1) {
            load_keys(now);
            next = pages_of(i + 8);
        }
        const bool full = ok[0] && ok[1] && j0 + 31 <= pf && (!a.window || j0 > pl - a.window || j0 + 31 < a.sinks);
        uint32_t vis = 0xFFu;
        bool seen = true, bad = false;
        float top = -INFINITY;
        if (!full) {
            vis = 0;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const int j = j0 + 16 * (n >> 2) + 4 * kq + (n & 3);
                if (ok[n >> 2] && sees(a, p, j)) vis |= 1u << n;
                // a key that no row sees counts for nothing, whatever lies there
                if (!(ok[n >> 2] && j <= pl && (!a.window || j > pf - a.window || j < a.sinks))) {
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int e = 0; e < VW / 2; e++) vv[n][b][e] = 0;
                }
                uint32_t inf = 0;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int e = 0; e < VW / 2; e++) {
                        const uint32_t y = vv[n][b][e] & (Op<E>::kExp * 0x10001u);
                        inf |= ((y & 0xFFFFu) == Op<E>::kExp) | ((y >> 16) == Op<E>::kExp);
                    }
                bad |= inf != 0;
                if (vis >> n & 1) top = fmaxf(top, s[n >> 2][n & 3]);
            }
            bad = __any(bad);
            const unsigned long long any = __ballot(vis != 0);
            seen = ((any >> li | any >> (16 + li) | any >> (32 + li) | any >> (48 + li)) & 1) != 0;
        } else {
#pragma unroll
            for (int n = 0; n < 8; n++) top = fmaxf(top, s[n >> 2][n & 3]);
        }
        top = max_x32(max_x16(top));
        const float high = seen ? fmaxf(ceilf(top * c), kLowest) : -INFINITY;
        const bool higher = high > m + Op<E>::kTol;
        if (__any(higher)) {
            const float mn = higher ? high : m, f = higher ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
            l *= f;
#pragma unroll
            for (int d = 0; d < D / 16; d++) o[d] *= f;
            m = mn;
        }
        float pr[8];
#pragma unroll
        for (int n = 0; n < 8; n++) {
            // (with 24 bits behind the exponential: a far exponent would round its argument)
            pr[n] = NP == 3 ? __builtin_amdgcn_exp2f(fmaf(s[n >> 2][n & 3], c, -m)) * raised : __builtin_amdgcn_exp2f(fmaf(s[n >> 2][n & 3], c, lift - m));
            if (!full && !(vis >> n & 1)) pr[n] = 0.f;
            l += pr[n];
        }
        V8<E> pp[NW];
        planes<E, NW>(pr, pp);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < VW; e++) {
                u32x4 t;
#pragma unroll
                for (int k = 0; k < 4; k++) t[k] = __builtin_amdgcn_perm(vv[2 * k + 1][b][e / 2], vv[2 * k][b][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
                f32x4 &acc = o[b * VW + e];
                if (bad) {   // values that are not finite make the rows that see them so, and no other (0 times infinity)
                    u32x4 mark, sight;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const bool lo = (t[k] & Op<E>::kExp) == Op<E>::kExp, hi = (t[k] >> 16 & Op<E>::kExp) == Op<E>::kExp;
                        mark[k] = (lo ? Op<E>::kOne : 0u) | (hi ? Op<E>::kOne << 16 : 0u);
                        t[k] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
                        sight[k] = (vis >> (2 * k) & 1 ? Op<E>::kOne : 0u) | (vis >> (2 * k + 1) & 1 ? Op<E>::kOne << 16 : 0u);
                    }
                    const f32x4 n = Op<E>::mfma16(__builtin_bit_cast(V8<E>, mark), __builtin_bit_cast(V8<E>, sight), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[k] += n[k] > 0.f ? NAN : 0.f;
                }
#pragma unroll
                for (int k = NW - 1; k >= 0; k--) acc = Op<E>::mfma16(__builtin_bit_cast(V8<E>, t), pp[k], acc);
            }
        if (i + 4 < i1) load_values(now);
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // ---- the four wavefronts' sums
    if (kq == 0) sm[w][li] = m, sl[w][li] = l;
    if (row < n_rows)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < VW; e += 4) {
                    const int d = b * VW + e;
                    *(f32x4 *)&so[w][li][16 * VW * b + VW * (4 * kq + r) + e] = f32x4{o[d][r], o[d + 1][r], o[d + 2][r], o[d + 3][r]};
                }
    __syncthreads();
    const int rt = tid >> 4, R0 = it.tile * 16 + rt;
    if (R0 >= n_rows) return;
    float mw[4], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        mw[k] = sm[k][rt];
        M = fmaxf(M, mw[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        mw[k] = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[k] - M);
        L += mw[k] * sl[k][rt];
    }
    const bool whole = it.pieces == 1;
    const float inv = M == -INFINITY ? 0.f : 1.f / L;   // a row that has seen nothing is 0
    const int t = token_of(a, R0), h = it.head * a.G + R0 - t * a.G, d0 = 4 * (tid & 15);
    const int64_t to = (int64_t)it.slot * 16 + rt;
    if (!whole && d0 == 0) *part_stat(a, to, 16, D) = float2{M, L};
    R *out = (R *)a.out + (it.s.start + t) * a.o_tok + (int64_t)h * D + d0;
    const R *gate = a.gate ? (const R *)a.gate + (it.s.start + t) * a.g_tok + h * a.g_head + d0 : nullptr;
#pragma unroll
    for (int d = 0; d < D; d += 64) {
        f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; k++) y += mw[k] * *(const f32x4 *)&so[k][rt][d0 + d];
        if (whole) finish4(y, inv, gate ? gate + d : nullptr, out + d);
        else *(f32x4 *)(part_sums(a, to, D) + d0 + d) = y;
    }
}

template <int D>
static void few(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    const dim3 grid((unsigned)items);
    if (!a.table) {
        if (a.type == kRowF16) attn_few_kernel<D, _Float16, 1, kRowF16, false><<<grid, 256, 0, st>>>(a);
        else attn_few_kernel<D, __bf16, 1, kRowBf16, false><<<grid, 256, 0, st>>>(a);
    } else if (a.type == kRowF16) attn_few_kernel<D, _Float16, 1, kRowF16, true><<<grid, 256, 0, st>>>(a);
    else if (a.type == kRowBf16) attn_few_kernel<D, __bf16, 1, kRowBf16, true><<<grid, 256, 0, st>>>(a);
    else if (a.kv_type == kRowF16) attn_few_kernel<D, _Float16, 2, kRowF32, true><<<grid, 256, 0, st>>>(a);
    else attn_few_kernel<D, __bf16, 3, kRowF32, true><<<grid, 256, 0, st>>>(a);
}
int attn_few_launch(const BatchAttnArgs &a, int64_t items, hipStream_t st) {
    if (a.D == 64) few<64>(a, items, st);
    else if (a.D == 128) few<128>(a, items, st);
    else few<256>(a, items, st);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ------------------------------------------------------------------- cut --

// The tiles of a piece (piece_of) of more than 64 requests, or that none is cut, as find_item finds them. Where every wavefront of the other kernels sums the
// requests for itself, 104 to 1000 requests of 100 positions take 7 to 126 us more; this launch and that of a join that finds nothing take 4 to 13.
template <int BM, int BN>
__global__ __launch_bounds__(1024) void attn_cut_kernel(const BatchAttnArgs a) {
    __shared__ float su[16];
    __shared__ int sn[16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    float u = 0.f;
    int most = 0;
    for (int r = tid; r < a.n_req; r += 1024) {
        const Seq s = seq_of<BM, BN>(a, r);
        u += (float)s.tiles * (float)s.len;
        most = max(most, s.len);
    }
    u = wave_sum(u);
    for (int o = 32; o; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    if (lane == 0) su[w] = u, sn[w] = most;
    __syncthreads();
    if (tid) return;
    for (int k = 1; k < 16; k++) {
        u += su[k];
        most = max(most, sn[k]);
    }
    const int per = piece_of(a, u);
    *a.per = most > 2 * (int64_t)per ? per : INT32_MAX;
}
int attn_cut_launch(const BatchAttnArgs &a, int BM, hipStream_t st) {
    if (BM == kFewRows) attn_cut_kernel<kFewRows, kFewKeys><<<1, 1024, 0, st>>>(a);
    else if (many_keys(a.D) == 32) attn_cut_kernel<kManyRows, 32><<<1, 1024, 0, st>>>(a);
    else attn_cut_kernel<kManyRows, 64><<<1, 1024, 0, st>>>(a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ----------------------------------------------------------------- merge --

// Rows in more than one piece, joined by D / 4 threads each. Of few rows there are many pieces: the work-group takes a row at a time, its threads'
// other runs the next pieces (128 pieces of a row of 256 dims 6 us, 23 by a wavefront a row). Of many rows there are few: the runs take the next rows.
template <int D, int BM, int BN, int RT>
__global__ __launch_bounds__(256) void attn_merge_kernel(const BatchAttnArgs a) {
    typedef typename Row<RT>::t R;
    constexpr int TD = D / 4, TP = 256 / TD;
    constexpr bool FEW = BM == kFewRows;
    __shared__ __align__(16) float so[FEW ? TP : 1][D];
    __shared__ float sl[TP];
    const int tid = threadIdx.x, lane = tid & 63, d = 4 * (tid % TD), tp = tid / TD;
    Item it;
    if (!find_item<BM, BN, true>(a, blockIdx.x, it)) return;
    const int n_rows = min(it.s.rows * a.G - it.tile * BM, BM);
    const int64_t step = (int64_t)a.Hkv * BM;
    for (int i = FEW ? blockIdx.y : blockIdx.y * TP + tp; i < n_rows; i += FEW ? (int)gridDim.y : (int)gridDim.y * TP) {   // FEW: the same for the whole work-group
        const int64_t at = (int64_t)it.slot * BM + i;
        float M = -INFINITY, L = 0.f;
        if (FEW) {
            for (int p = lane; p < it.pieces; p += 64) M = fmaxf(M, part_stat(a, at + p * step, BM, D)->x);
            M = xjd::wave_max(M);
        } else {
#pragma unroll 4
            for (int p = 0; p < it.pieces; p++) M = fmaxf(M, part_stat(a, at + p * step, BM, D)->x);
        }
        f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
        if (M != -INFINITY)
#pragma unroll 4
            for (int p = FEW ? tp : 0; p < it.pieces; p += FEW ? TP : 1) {
                const float2 s = *part_stat(a, at + p * step, BM, D);
                const f32x4 x = *(const f32x4 *)(part_sums(a, at + p * step, D) + d);
                const float f = __builtin_amdgcn_exp2f(s.x - M);
                L += f * s.y;
                y += f * x;
            }
        if constexpr (FEW) {
            *(f32x4 *)&so[tp][d] = y;
            if (d == 0) sl[tp] = L;
            __syncthreads();
            if (tp == 0)
#pragma unroll
                for (int k = 1; k < TP; k++) {
                    y += *(const f32x4 *)&so[k][d];
                    L += sl[k];
                }
            __syncthreads();
            if (tp) continue;
        }
        const int row = it.tile * BM + i, t = token_of(a, row), h = it.head * a.G + row - t * a.G;
        finish4(y, M == -INFINITY ? 0.f : 1.f / L, a.gate ? (const R *)a.gate + (it.s.start + t) * a.g_tok + h * a.g_head + d : nullptr,
                (R *)a.out + (it.s.start + t) * a.o_tok + (int64_t)h * D + d);
    }
}
template <int D, int BM, int BN>
static void merge(const BatchAttnArgs &a, dim3 grid, hipStream_t st) {
    if (a.type == kRowF32) attn_merge_kernel<D, BM, BN, kRowF32><<<grid, 256, 0, st>>>(a);
    else if (a.type == kRowF16) attn_merge_kernel<D, BM, BN, kRowF16><<<grid, 256, 0, st>>>(a);
    else attn_merge_kernel<D, BM, BN, kRowBf16><<<grid, 256, 0, st>>>(a);
}
template <int BM, int D>
static void merge(const BatchAttnArgs &a, dim3 grid, hipStream_t st) {
    if constexpr (BM == kFewRows) merge<D, BM, kFewKeys>(a, grid, st);
    else merge<D, BM, many_keys(D)>(a, grid, st);
}
int attn_merge_launch(const BatchAttnArgs &a, int BM, int64_t groups, bool rare, hipStream_t st) {
    // Of few rows as many work-groups a tile as it has rows, as far as that is known: each has to find its tile. Of many rows one for 8 KB of its sums, for four times
    // that where a batch may have so many tiles that a cut is rare (8200 rows of 32 heads on 8 of 128, uncut: 564 us, 573 with all of them, 561 without a join).
    const int known = a.max_new > 0 ? a.max_new : 2;
    const dim3 grid((unsigned)groups, BM == kFewRows ? (int)std::min<int64_t>(BM, (int64_t)known * a.G) : BM * a.D / (rare ? 4096 : 1024));
    if (BM == kFewRows) {
        if (a.D == 64) merge<kFewRows, 64>(a, grid, st);
        else if (a.D == 128) merge<kFewRows, 128>(a, grid, st);
        else merge<kFewRows, 256>(a, grid, st);
    } else {
        if (a.D == 64) merge<kManyRows, 64>(a, grid, st);
        else if (a.D == 128) merge<kManyRows, 128>(a, grid, st);
        else merge<kManyRows, 256>(a, grid, st);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace xjk
