// Rotary positions with scaled frequencies (gfx950): xjh_rope_scaled.
//
// A pair (a, b) of a token at position p becomes (a c - b s, a s + b c) with
// c, s = mscale * cos, sin of p f_i. The angle is formed in turns in double, whole
// turns are dropped exactly, and sine and cosine of the rest are taken in float:
// an angle keeps 2^-24 of a turn at any position (a float product p f_i loses it at
// once: 2^-8 of a radian at 100000).
#include "common.h"
#include "kernels.h"

namespace xjk {

// One work-group per token: the token's cosines and sines once in LDS, then every
// head's pairs and, when the result goes elsewhere, the elements that do not turn.
__global__ __launch_bounds__(256) void rope_scaled_kernel(const RopeArgs a) {
    __shared__ float2 cs[kRopeMaxPairs];
    const int t = blockIdx.x, tid = threadIdx.x, half = a.n_rot / 2;
    const double p = a.pos ? a.pos[t] : (double)a.pos0 + t;
    if (tid < half) {
        const double w = p * a.f[tid];
        float s, c;
        sincospif((float)(2.0 * (w - rint(w))), &s, &c);
        cs[tid] = float2{c * a.mscale, s * a.mscale};
    }
    __syncthreads();
    const float *xt = a.x + t * a.x_tok;
    float *ot = a.out + t * a.o_tok;
    for (int i = tid; i < a.n_heads * half; i += 256) {
        const int h = i / half, j = i % half;
        const int e0 = a.interleaved ? 2 * j : j, e1 = a.interleaved ? 2 * j + 1 : j + half;
        const float u = xt[h * a.x_head + e0], v = xt[h * a.x_head + e1];
        ot[h * a.o_head + e0] = u * cs[j].x - v * cs[j].y;
        ot[h * a.o_head + e1] = u * cs[j].y + v * cs[j].x;
    }
    if (a.out == a.x) return;
    const int rest = a.D - a.n_rot;
    for (int i = tid; i < a.n_heads * rest; i += 256) {
        const int h = i / rest, j = a.n_rot + i % rest;
        ot[h * a.o_head + j] = xt[h * a.x_head + j];
    }
}

int rope_scaled_launch(const RopeArgs &a, hipStream_t st) {
    if (a.T < 1 || a.n_heads < 1 || a.n_rot < 2 || a.n_rot % 2 || a.n_rot / 2 > kRopeMaxPairs || a.n_rot > a.D) return -1;
    hipLaunchKernelGGL(rope_scaled_kernel, dim3(a.T), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace xjk
