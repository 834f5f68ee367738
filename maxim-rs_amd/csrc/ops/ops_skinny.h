// Products of few rows (a token or a few at a time): the weights are read once
// and bound them.
//
// A block takes 16 columns of C and all of k, its eight waves an eighth of k
// each: a wave brings 16 rows of the weights, 16 bytes a lane, straight from
// memory into the matrix cores' operand registers, eight loads ahead of their
// use, and the rows of A likewise from the caches. The waves' sums are added
// in LDS, so no partial sums go through memory and there is one launch.
// (4096 x 4096 bf16 weights: 9.0 us for one row, 3.7 TB/s, 10.6 us for 16; as
// 64 x 64 tiles, cut and joined, 11.6 and 11.4. With two blocks of rows a wave
// 17 rows took 14.7 us, the tiles 12.1.) Where k is long and the columns few
// the card stands idle: plan_product (exec/ops.cpp) has the rule, and both sides.
#pragma once

#include "ops_gemm.h"

template <typename T>
__device__ __forceinline__ void gemm_skinny(const OpsGemmArgs &g) {
    constexpr int E = 16 / sizeof(T), STEP = 4 * E, W = 8, AHEAD = 8;
    typedef typename Mma<T>::Frag Frag;
    __shared__ f32x4 sums[W][64];
    const float back = back_of<T>(g);
    const int t = threadIdx.x, l = t & 63, w = t >> 6, r = l & 15, q = l >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    // this wave's k's, whole steps; past them nothing is loaded
    const int each = (g.k + W * STEP - 1) / (W * STEP) * STEP, kbeg = w * each + q * E, kend = min(g.k, (w + 1) * each);
    const T *b = static_cast<const T *>(g.b) + min(n0 + r, (int64_t)g.n - 1) * g.ldb;
    const T *a = static_cast<const T *>(g.a) + (int64_t)min(r, g.m - 1) * g.lda;
    f32x4 acc = {0, 0, 0, 0};
    // rows past the last are the last again: their sums are not stored
    const int steps = each / STEP, whole = max(0, (kend - w * each)) / STEP;
    auto go = [&](const Vec<T, E> &fb, const Vec<T, E> &fa) {
        acc = Mma<T>::go(__builtin_bit_cast(Frag, fb), __builtin_bit_cast(Frag, fa), acc);
    };
    int s = 0;
    for (; s + AHEAD <= whole; s += AHEAD) {
        Vec<T, E> fb[AHEAD], fa[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int k = kbeg + (s + j) * STEP;
            fb[j] = load_n<T, E>(b + k);
            fa[j] = load_n<T, E>(a + k);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) go(fb[j], fa[j]);
    }
    for (; s < steps; ++s) {
        const int k = kbeg + s * STEP;
        go(load_upto<T, E>(b + k, kend - k), load_upto<T, E>(a + k, kend - k));
    }
    sums[w][l] = acc;
    __syncthreads();
    if (t >= 64) return;
    // lane l: row l % 16, columns 4 (l / 16) + 0..3
    f32x4 v = sums[0][l];
#pragma unroll
    for (int k = 1; k < W; ++k) v += sums[k][l];
    const int64_t m = r, n = n0 + q * 4;
    float out[4] = {v[0], v[1], v[2], v[3]}, bias[4];
    Extra<T, 4> x;
    bias_fetch<T, 4>(g, n, bias);
    extra_fetch<T, 4>(g, m, n, x);
    gemm_finish<T, 4>(g, m, n, out, bias, x, back);
}

#define OPS_SKINNY(name, T) \
    extern "C" __global__ __launch_bounds__(512) void mxo_skinny_##name(OpsGemmArgs g) { gemm_skinny<T>(g); }

OPS_SKINNY(bf16, bf16)
OPS_SKINNY(f16, f16)
OPS_SKINNY(f32, float)
