// LayerNorm, its backward pass and the activation's derivative with the
// bias's gradient: passes over [rows][cols] activations of either order.
#pragma once

#include "ops_common.h"

// Sum over a block of 1024 threads, in every thread; `at` holds 16 floats.
__device__ __forceinline__ float block_sum(float v, float *at) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += at[i];
    return s;
}

// Any shape and order: a block of 1024 threads a row, three passes over it.
template <typename T>
__device__ __forceinline__ void ln_any(const OpsLnArgs &a) {
    __shared__ float at[16];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.xrs;
        T *y = static_cast<T *>(a.y) + r * a.yrs;
        float s = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) s += to_f<T>(x[c * a.xcs]);
        const float mean = block_sum(s, at) / (float)a.cols;
        s = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float d = to_f<T>(x[c * a.xcs]) - mean;
            s += d * d;
        }
        const float rstd = 1.0f / sqrtf(block_sum(s, at) / (float)a.cols + a.eps);
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float d = (to_f<T>(x[c * a.xcs]) - mean) * rstd;
            const float b = a.bias ? param<T>(a.bias, c, a.param_f32) : 0.0f;
            y[c * a.ycs] = from_f<T>(d * param<T>(a.scale, c, a.param_f32) + b);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__device__ __forceinline__ void ln_bwd_any(const OpsLnBwdArgs &a) {
    __shared__ float at[16];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.xrs;
        const T *dy = static_cast<const T *>(a.dy) + r * a.dyrs;
        const T *add = a.add ? static_cast<const T *>(a.add) + r * a.ars : nullptr;
        T *dx = static_cast<T *>(a.dx) + r * a.dxrs;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s = 0.0f, q = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float gr = to_f<T>(dy[c * a.dycs]) * param<T>(a.scale, c, a.param_f32);
            s += gr;
            q += gr * ((to_f<T>(x[c * a.xcs]) - mean) * rstd);
        }
        s = block_sum(s, at) / (float)a.cols;
        q = block_sum(q, at) / (float)a.cols;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float gr = to_f<T>(dy[c * a.dycs]) * param<T>(a.scale, c, a.param_f32);
            const float xh = (to_f<T>(x[c * a.xcs]) - mean) * rstd;
            float v = rstd * (gr - s - xh * q);
            if (add) v += to_f<T>(add[c * a.acs]);
            dx[c * a.dxcs] = from_f<T>(v);
        }
    }
}

// dscale's and dbias's partial sums, 64 columns by a run of rows a block.
template <typename T>
__device__ __forceinline__ void ln_param_any(const OpsLnBwdArgs &a) {
    __shared__ float sh[2][4][64];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + l, p = blockIdx.y;
    const int64_t chunk = (a.rows + a.nparts - 1) / a.nparts, end = min(a.rows, (p + 1) * chunk);
    float s = 0.0f, b = 0.0f;
    if (c < a.cols)
        for (int64_t r = p * chunk + w; r < end; r += 4) {
            const float dy = to_f<T>(static_cast<const T *>(a.dy)[r * a.dyrs + c * a.dycs]);
            const float xh = (to_f<T>(static_cast<const T *>(a.x)[r * a.xrs + c * a.xcs]) - a.mean[r]) * a.rstd[r];
            s += dy * xh;
            b += dy;
        }
    sh[0][w][l] = s;
    sh[1][w][l] = b;
    __syncthreads();
    if (w < 2 && c < a.cols)
        a.part[(p * 2 + w) * a.cols + c] = (sh[w][0][l] + sh[w][1][l]) + (sh[w][2][l] + sh[w][3][l]);
}

// dz and the bias's partial sums, 64 columns by a run of rows a block.
template <typename T>
__device__ __forceinline__ void dz_any(const OpsDzArgs &a) {
    __shared__ float sh[4][64];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + l, p = blockIdx.y;
    const int64_t chunk = (a.rows + a.nparts - 1) / a.nparts, end = min(a.rows, (p + 1) * chunk);
    float s = 0.0f;
    if (c < a.cols)
        for (int64_t r = p * chunk + w; r < end; r += 4) {
            float v = to_f<T>(static_cast<const T *>(a.dy)[r * a.dyrs + c * a.dycs]);
            if (a.z) v *= act_bwd(a.act, a.slope, to_f<T>(static_cast<const T *>(a.z)[r * a.zrs + c * a.zcs]));
            if (a.dz) static_cast<T *>(a.dz)[r * a.drs + c * a.dcs] = from_f<T>(v);
            s += v;
        }
    if (!a.part) return;
    sh[w][l] = s;
    __syncthreads();
    if (w == 0 && c < a.cols) a.part[p * a.cols + c] = (sh[0][l] + sh[1][l]) + (sh[2][l] + sh[3][l]);
}

// Partial sums added in a fixed order: 16 rows of 64 columns a block, each
// wave a sixteenth of the parts, then the waves' sums.
__device__ __forceinline__ void join_store(void *out, int dtype, int64_t i, float v) {
    if (dtype == MXO_F32) static_cast<float *>(out)[i] = v;
    else if (dtype == MXO_F16) static_cast<f16 *>(out)[i] = from_f<f16>(v);
    else static_cast<bf16 *>(out)[i] = from_f<bf16>(v);
}
extern "C" __global__ __launch_bounds__(1024) void mxo_join_parts(OpsJoinArgs a) {
    __shared__ float sh[16][64];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, which = blockIdx.y;
    const int64_t c = (int64_t)blockIdx.x * 64 + l;
    float s = 0.0f;
    if (c < a.n)
        for (int p = w; p < a.nparts; p += 16) s += a.part[((int64_t)p * a.nout + which) * a.n + c];
    sh[w][l] = s;
    __syncthreads();
    if (w || c >= a.n) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sh[i][l];
    join_store(which ? a.out1 : a.out0, a.dtype, c, s);
}

#define OPS_ROWS_TYPE(name, T)                                                                                        \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_any_##name(OpsLnArgs a) { ln_any<T>(a); }               \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_bwd_any_##name(OpsLnBwdArgs a) { ln_bwd_any<T>(a); }    \
    extern "C" __global__ __launch_bounds__(256) void mxo_ln_param_any_##name(OpsLnBwdArgs a) { ln_param_any<T>(a); } \
    extern "C" __global__ __launch_bounds__(256) void mxo_dz_any_##name(OpsDzArgs a) { dz_any<T>(a); }

OPS_ROWS_TYPE(bf16, bf16)
OPS_ROWS_TYPE(f16, f16)
OPS_ROWS_TYPE(f32, float)
