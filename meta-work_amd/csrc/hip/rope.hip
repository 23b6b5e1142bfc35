// Rotary positions with scaled frequencies (gfx950): xjh_rope_scaled.
//
// A pair (a, b) of a token at position p becomes (a c - b s, a s + b c) with
// c, s = mscale * cos, sin of p f_i. The angle is formed in turns in double, whole
// turns are dropped exactly, and sine and cosine of the rest are taken in float:
// an angle keeps 2^-24 of a turn at any position (a float product p f_i loses it at
// once: 2^-8 of a radian at 100000).
// Bound by the rows' bytes (4096 tokens of 16 heads of 256: 134 MB in 26.9 us, 5.0 TB/s; a 1 GiB copy reaches 5.15); one
// token's 2.7 us are a launch.
#include "common.h"
#include "kernels.h"

namespace xjk {

constexpr int kRopeGridX = 1 << 23;   // (a grid's dimension times 256 threads stays below 2^32)

// One work-group per token: the token's cosines and sines once in LDS, then every
// head's pairs and, when the result goes elsewhere, the elements that do not turn.
// V: elements per access, 4 where every run of them (a half of n_rot, n_rot, the
// rest of the head) is a multiple of 4 (with 1: those 4096 tokens, interleaved, 30.4 us, one token 4.4).
template <int V>
__global__ __launch_bounds__(256) void rope_scaled_kernel(const RopeArgs a) {
    typedef float vec __attribute__((ext_vector_type(V)));
    typedef float vec_u __attribute__((ext_vector_type(V), aligned(4)));
    __shared__ __align__(16) float cs[2][kRopeMaxPairs];
    const int64_t t = (int64_t)blockIdx.y * kRopeGridX + blockIdx.x;
    const int tid = threadIdx.x, half = a.n_rot / 2;
    if (t >= a.T) return;
    const double p = a.pos ? a.pos[t] : (double)a.pos0 + t;
    if (tid < half) {
        const double w = p * a.f[tid];
        float s, c;
        sincospif((float)(2.0 * (w - rint(w))), &s, &c);
        cs[0][tid] = c * a.mscale;
        cs[1][tid] = s * a.mscale;
    }
    __syncthreads();
    const float *xt = a.x + t * a.x_tok;
    float *ot = a.out + t * a.o_tok;
    if (a.interleaved) {   // V pairs are 2 V elements
        for (int i = tid; i < a.n_heads * (half / V); i += 256) {
            const int h = i / (half / V), j = i % (half / V) * V;
            const vec x0 = *(const vec_u *)(xt + h * a.x_head + 2 * j), x1 = *(const vec_u *)(xt + h * a.x_head + 2 * j + V);
            vec y[2];
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float u = V == 1 ? x0[0] : k < V / 2 ? x0[2 * k % V] : x1[2 * k % V], v = V == 1 ? x1[0] : k < V / 2 ? x0[(2 * k + 1) % V] : x1[(2 * k + 1) % V];
                const float c = cs[0][j + k], s = cs[1][j + k];
                y[2 * k / V][2 * k % V] = u * c - v * s;
                y[(2 * k + 1) / V][(2 * k + 1) % V] = u * s + v * c;
            }
            *(vec_u *)(ot + h * a.o_head + 2 * j) = y[0];
            *(vec_u *)(ot + h * a.o_head + 2 * j + V) = y[1];
        }
    } else {
        for (int i = tid; i < a.n_heads * (half / V); i += 256) {
            const int h = i / (half / V), j = i % (half / V) * V;
            const vec u = *(const vec_u *)(xt + h * a.x_head + j), v = *(const vec_u *)(xt + h * a.x_head + j + half);
            const vec c = *(const vec *)&cs[0][j], s = *(const vec *)&cs[1][j];
            *(vec_u *)(ot + h * a.o_head + j) = u * c - v * s;
            *(vec_u *)(ot + h * a.o_head + j + half) = u * s + v * c;
        }
    }
    const int rest = (a.D - a.n_rot) / V;
    if (a.out == a.x || !rest) return;
    for (int i = tid; i < a.n_heads * rest; i += 256) {
        const int h = i / rest, j = a.n_rot + i % rest * V;
        *(vec_u *)(ot + h * a.o_head + j) = *(const vec_u *)(xt + h * a.x_head + j);
    }
}

int rope_scaled_launch(const RopeArgs &a, hipStream_t st) {
    if (a.T < 1 || a.n_heads < 1 || a.n_rot < 2 || a.n_rot % 2 || a.n_rot / 2 > kRopeMaxPairs || a.n_rot > a.D) return -1;
    const bool v4 = a.n_rot % 8 == 0 && (a.out == a.x || (a.D - a.n_rot) % 4 == 0);
    const dim3 grid(a.T < kRopeGridX ? a.T : kRopeGridX, (a.T - 1) / kRopeGridX + 1);
    if (v4) hipLaunchKernelGGL(rope_scaled_kernel<4>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(rope_scaled_kernel<1>, grid, dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace xjk
