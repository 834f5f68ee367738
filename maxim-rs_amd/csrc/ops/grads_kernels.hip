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
__device__ __forceinline__ double chunk_squares(const T *p, int64_t have, int t) {
    constexpr int E = 16 / sizeof(T);
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

__device__ __forceinline__ double wave_sum(double s) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
    return s;
}
__device__ __forceinline__ double block_sum(double s, double *at) {
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = s;
    __syncthreads();
    return (at[0] + at[1]) + (at[2] + at[3]);
}

// Chunk c of the list: its tensor's place, elements and type.
struct Chunk {
    int tensor, type;
    int64_t at, have;
};
__device__ __forceinline__ Chunk chunk_at(const GradsArgs &a, uint32_t lo, uint32_t hi, uint32_t c) {
    const int i = tensor_of(a, lo, hi, c), type = (int)(a.n[i] >> 56);
    const int64_t at = (int64_t)(c - a.first[i]) * (MXN_CHUNK / (type == MXO_F32 ? 4 : 2));
    return {i, type, at, (int64_t)(a.n[i] & ~(0xffull << 56)) - at};
}
// The sum of its squares, 256 threads' parts.
__device__ __forceinline__ double squares_of(const GradsArgs &a, const Chunk &c, int t) {
    const void *p = a.src[c.tensor];
    if (c.type == MXO_F32) return chunk_squares<float>(static_cast<const float *>(p) + c.at, c.have, t);
    if (c.type == MXO_F16) return chunk_squares<f16>(static_cast<const f16 *>(p) + c.at, c.have, t);
    return chunk_squares<bf16>(static_cast<const bf16 *>(p) + c.at, c.have, t);
}

extern "C" __global__ __launch_bounds__(256) void mxn_squares(GradsArgs a) {
    __shared__ double at[4];
    const int l = threadIdx.x & 63;
    const uint32_t lo = first_of(a, l), hi = first_of(a, l + 64), chunks = a.first[a.count];
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) s += squares_of(a, chunk_at(a, lo, hi, c), threadIdx.x);
    s = block_sum(s, at);
    if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

// The blocks' sums, in a fixed order.
extern "C" __global__ __launch_bounds__(256) void mxn_norm(GradsJoinArgs a) {
    __shared__ double at[4];
    double s = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.nparts; i += 256) s += a.part[i];
    s = block_sum(s, at);
    if (threadIdx.x == 0) *a.norm = (float)__builtin_sqrt(s);
}

// What gradients are multiplied by: a norm that is not finite, or not past the
// bound, leaves them as they are. A quotient below fp32's normal range has too few
// bits of its own, and a gradient near the range's other end brings its product
// back: there it is 64 bits wide.
struct Factor {
    float f;
    double wide;  // not 0: instead of f
};
__device__ __forceinline__ Factor factor(float norm, float most) {
    if (!(norm > most && norm < __builtin_inff())) return {1.0f, 0.0};
    const float f = most / norm;
    return {f, f < 0x1p-126f ? (double)most / norm : 0.0};
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T *p, T *q, int64_t have, const Factor &f, int t) {
    constexpr int E = 16 / sizeof(T);
    auto scale = [&](Vec<T, E> &v) {
        if (f.f == 1.0f) return;  // the same bits, NaN's too
        if (f.wide != 0.0) {
#pragma unroll
            for (int e = 0; e < E; ++e) v.v[e] = from_f<T>((float)(to_f<T>(v.v[e]) * f.wide));
            return;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) v.v[e] = from_f<T>(to_f<T>(v.v[e]) * f.f);
    };
    if (have >= MXN_CHUNK / (int)sizeof(T)) {
        Vec<T, E> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = load_n<T, E>(p + (u * 256 + t) * E);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            scale(v[u]);
            store_out<T, E>(q + (u * 256 + t) * E, v[u], E);
        }
    } else {
        for (int k = t * E; k < have; k += 256 * E) {
            Vec<T, E> v = load_upto<T, E>(p + k, have - k);
            scale(v);
            store_upto<T, E>(q + k, v, have - k);
        }
    }
}

__device__ __forceinline__ void scale_chunk(const GradsArgs &a, const Chunk &c, const Factor &f, int t) {
    const void *p = a.src[c.tensor];
    void *q = a.dst[c.tensor];
    if (f.f == 1.0f && p == q) return;
    if (c.type == MXO_F32)
        chunk_scale<float>(static_cast<const float *>(p) + c.at, static_cast<float *>(q) + c.at, c.have, f, t);
    else if (c.type == MXO_F16)
        chunk_scale<f16>(static_cast<const f16 *>(p) + c.at, static_cast<f16 *>(q) + c.at, c.have, f, t);
    else
        chunk_scale<bf16>(static_cast<const bf16 *>(p) + c.at, static_cast<bf16 *>(q) + c.at, c.have, f, t);
}

extern "C" __global__ __launch_bounds__(256) void mxn_clip(GradsArgs a) {
    const int l = threadIdx.x & 63;
    const uint32_t lo = first_of(a, l), hi = first_of(a, l + 64), chunks = a.first[a.count];
    const Factor f = factor(*a.norm, a.max_norm);
    for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) scale_chunk(a, chunk_at(a, lo, hi, chunks - 1 - b), f, threadIdx.x);
}

// A list of few chunks in one block and one launch, four chunks at a time. (The
// gradients of a 64-channel block, six tensors, in seven chunks: three launches
// 3.7, 1.8 and 3.7 us and 30 us a call from Python, this 4.9 and 21.)
extern "C" __global__ __launch_bounds__(1024) void mxn_small(GradsArgs a) {
    __shared__ double at[4][4];
    const int l = threadIdx.x & 63, t = threadIdx.x & 255, g = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const uint32_t lo = first_of(a, l), hi = first_of(a, l + 64), chunks = a.first[a.count];
    double s = 0.0;
    for (uint32_t c = g; c < chunks; c += 4) s += squares_of(a, chunk_at(a, lo, hi, c), t);
    s = wave_sum(s);
    if (l == 0) at[g][t >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += (at[i][0] + at[i][1]) + (at[i][2] + at[i][3]);
    const float norm = (float)__builtin_sqrt(s);
    if (threadIdx.x == 0) *a.norm = norm;
    if (!a.clip) return;
    const Factor f = factor(norm, a.max_norm);
    for (uint32_t c = g; c < chunks; c += 4) scale_chunk(a, chunk_at(a, lo, hi, c), f, t);
}
