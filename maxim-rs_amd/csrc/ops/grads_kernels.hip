// The gfx950 code object of the gradients' global norm and clipping
// (include/maxim_block_ops.h).
//
// Both walk over a list of tensors in chunks of 16 KiB, 16 bytes a lane and
// four loads in flight, any alignment; a block finds a chunk's tensor by
// comparing its number with 64 tensors' first chunks at once. Bound by memory:
// the norm reads everything once, clipping reads it again and writes it, last
// chunks first, since the norm has just read those and the 256 MB cache may
// still hold them.
#include "grads_args.h"
#include "ops_common.h"

// The tensor of chunk c: the last whose first chunk is not past it (an empty
// tensor has none of its own).
__device__ __forceinline__ int tensor_of(const GradsArgs &a, uint32_t lo, uint32_t hi, uint32_t c) {
    return __builtin_popcountll(__builtin_amdgcn_ballot_w64(lo <= c)) +
           __builtin_popcountll(__builtin_amdgcn_ballot_w64(hi <= c)) - 1;
}
__device__ __forceinline__ uint32_t first_of(const GradsArgs &a, int i) {
    return i < a.count ? a.first[i] : 0xffffffffu;
}

// The squares of fp32 values reach from 2^-298 to 2^256, and a model has more
// elements than fp32 sums keep: they are formed and added in 64 bits.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T *p, int64_t have) {
    constexpr int E = 16 / sizeof(T);
    const int t = threadIdx.x;
    double s = 0.0;
    if (have >= MXN_CHUNK / (int)sizeof(T)) {
        Vec<T, E> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = load_n<T, E>(p + (u * 256 + t) * E);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double d = to_f<T>(v[u].v[e]);
                s = __builtin_fma(d, d, s);
            }
    } else {
        for (int k = t * E; k < have; k += 256 * E) {
            const Vec<T, E> v = load_upto<T, E>(p + k, have - k);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double d = to_f<T>(v.v[e]);
                s = __builtin_fma(d, d, s);
            }
        }
    }
    return s;
}

__device__ __forceinline__ double block_sum(double s, double *at) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = s;
    __syncthreads();
    return (at[0] + at[1]) + (at[2] + at[3]);
}

__device__ __forceinline__ void store_norm(float *norm, double s) { *norm = (float)__builtin_sqrt(s); }

extern "C" __global__ __launch_bounds__(256) void mxn_squares(GradsArgs a) {
    __shared__ double at[4];
    const int l = threadIdx.x & 63;
    const uint32_t lo = first_of(a, l), hi = first_of(a, l + 64), chunks = a.first[a.count];
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int i = tensor_of(a, lo, hi, c);
        const uint64_t n = a.n[i] & ~(0xffull << 56);
        const int type = (int)(a.n[i] >> 56);
        const int64_t k = (int64_t)(c - a.first[i]) * (MXN_CHUNK / (type == MXO_F32 ? 4 : 2)), have = (int64_t)n - k;
        if (type == MXO_F32) s += chunk_squares<float>(static_cast<const float *>(a.src[i]) + k, have);
        else if (type == MXO_F16) s += chunk_squares<f16>(static_cast<const f16 *>(a.src[i]) + k, have);
        else s += chunk_squares<bf16>(static_cast<const bf16 *>(a.src[i]) + k, have);
    }
    s = block_sum(s, at);
    if (threadIdx.x) return;
    // the only block of the only launch has the whole sum
    if (a.norm) store_norm(a.norm, s);
    else a.part[blockIdx.x] = s;
}

// The blocks' sums, in a fixed order.
extern "C" __global__ __launch_bounds__(256) void mxn_norm(GradsJoinArgs a) {
    __shared__ double at[4];
    double s = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.nparts; i += 256) s += a.part[i];
    s = block_sum(s, at);
    if (threadIdx.x == 0) store_norm(a.norm, s);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T *p, T *q, int64_t have, float f) {
    constexpr int E = 16 / sizeof(T);
    const int t = threadIdx.x;
    auto scale = [&](Vec<T, E> &v) {
        if (f == 1.0f) return;  // the same bits, NaN's too
#pragma unroll
        for (int e = 0; e < E; ++e) v.v[e] = from_f<T>(to_f<T>(v.v[e]) * f);
    };
    if (have >= MXN_CHUNK / (int)sizeof(T)) {
        Vec<T, E> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = load_n<T, E>(p + (u * 256 + t) * E);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            scale(v[u]);
            store_n<T, E>(q + (u * 256 + t) * E, v[u]);
        }
    } else {
        for (int k = t * E; k < have; k += 256 * E) {
            Vec<T, E> v = load_upto<T, E>(p + k, have - k);
            scale(v);
            store_upto<T, E>(q + k, v, have - k);
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void mxn_clip(GradsArgs a) {
    const int l = threadIdx.x & 63;
    const uint32_t lo = first_of(a, l), hi = first_of(a, l + 64), chunks = a.first[a.count];
    // a norm that is not finite, or none past the bound: as they are
    const float norm = *a.norm;
    const float f = norm > a.max_norm && norm < __builtin_inff() ? a.max_norm / norm : 1.0f;
    for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) {
        const uint32_t c = chunks - 1 - b;
        const int i = tensor_of(a, lo, hi, c);
        if (f == 1.0f && a.src[i] == a.dst[i]) continue;
        const uint64_t n = a.n[i] & ~(0xffull << 56);
        const int type = (int)(a.n[i] >> 56);
        const int64_t k = (int64_t)(c - a.first[i]) * (MXN_CHUNK / (type == MXO_F32 ? 4 : 2)), have = (int64_t)n - k;
        if (type == MXO_F32)
            chunk_scale<float>(static_cast<const float *>(a.src[i]) + k, static_cast<float *>(a.dst[i]) + k, have, f);
        else if (type == MXO_F16)
            chunk_scale<f16>(static_cast<const f16 *>(a.src[i]) + k, static_cast<f16 *>(a.dst[i]) + k, have, f);
        else
            chunk_scale<bf16>(static_cast<const bf16 *>(a.src[i]) + k, static_cast<bf16 *>(a.dst[i]) + k, have, f);
    }
}
