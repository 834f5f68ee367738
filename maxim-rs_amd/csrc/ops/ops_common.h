// Device helpers of the training and serving operators.
#pragma once

#include "../hip/common.h"
#include "ops_args.h"

typedef _Float16 f16;
typedef __bf16 bf16;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    return (float)v;
}
// Rounds to nearest even, as every store of a result does.
template <typename T>
__device__ __forceinline__ T from_f(float v) {
    return (T)v;
}

// N consecutive elements at any alignment of the element: the memory system
// takes unaligned vector accesses, so one load serves every row stride.
template <typename T, int N>
struct Vec {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_n(const T *p) {
    Vec<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T *p, const Vec<T, N> &v) {
    __builtin_memcpy(p, &v, sizeof(v));
}
// The first `have` of them (any number), the others zero.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_upto(const T *p, int64_t have) {
    if (have >= N) return load_n<T, N>(p);
    Vec<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = i < have ? p[i] : (T)0.0f;
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_upto(T *p, const Vec<T, N> &v, int64_t have) {
    if (have >= N) {
        store_n<T, N>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < have) p[i] = v.v[i];
}

// E elements at p, of which the first `have` are the operand's and the others
// anything, for the user to leave out (left out here, a load ahead of its use
// would be waited for). WHOLE: all of them or none (the extent is a multiple of E). A lane
// without any loads at `any`, which are the operand's too, and drops them. A
// lane with some loads E all the same where that stays inside the operand, up
// to its last E elements at `last`: at the ends of all rows but the last few.
// So only a wave there takes a branch, and loads are not waited for one by one.
template <typename T, int E, bool WHOLE>
__device__ __forceinline__ u32x4 load_raw(const T *p, const T *any, const T *last, int64_t have) {
    static_assert(E * sizeof(T) == 16, "");
    u32x4 w;
    if (!WHOLE && __builtin_amdgcn_ballot_w64((have > 0 ? p : any) > last) != 0)
        w = __builtin_bit_cast(u32x4, load_upto<T, E>(p, have));
    else
        __builtin_memcpy(&w, have > 0 ? p : any, 16);
    return w;
}
// The same with zeros past the first `have`. (Dropped by whole registers:
// element by element a 16-bit vector would be held in eight of them.)
template <typename T, int E, bool WHOLE>
__device__ __forceinline__ u32x4 load_in(const T *p, const T *any, const T *last, int64_t have) {
    u32x4 w = load_raw<T, E, WHOLE>(p, any, last, have);
    const int h = (int)min(have, (int64_t)E);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (WHOLE) w[i] = have > 0 ? w[i] : 0u;
        else if (sizeof(T) == 2) w[i] = h > 2 * i + 1 ? w[i] : h == 2 * i + 1 ? w[i] & 0xffffu : 0u;
        else w[i] = h > i ? w[i] : 0u;
    }
    return w;
}
template <typename T, int E, bool WHOLE>
__device__ __forceinline__ void store_in(T *p, const Vec<T, E> &v, int64_t have) {
    if constexpr (WHOLE) {
        if (have > 0) store_n<T, E>(p, v);
    } else {
        store_upto<T, E>(p, v, have);
    }
}

// 16 bytes of elements as they lie, converted where they are used: taken apart,
// a 16-bit vector would be held in eight registers instead of four.
template <typename T>
__device__ __forceinline__ float elem(const u32x4 &w, int e) {
    if constexpr (sizeof(T) == 4) {
        const uint32_t u = w[e];  // (of the vector's element itself the cast takes the first one)
        return __builtin_bit_cast(float, u);
    } else if constexpr (__is_same(T, bf16)) {
        return __builtin_bit_cast(float, e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    } else {
        return (float)__builtin_bit_cast(f16, (uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu));
    }
}
// The same value, of which the compiler keeps nothing that it worked out before:
// elements are converted again from here on.
__device__ __forceinline__ void reread(u32x4 &w) { asm volatile("" : "+v"(w)); }

// The same number, of which nothing is worked out before this place.
__device__ __forceinline__ int64_t here(int64_t v) {
    asm volatile("" : "+s"(v));
    return v;
}

// A parameter vector's element, of the activations' type or fp32.
template <typename T>
__device__ __forceinline__ float param(const void *p, int64_t i, int f32) {
    return f32 ? static_cast<const float *>(p)[i] : to_f<T>(static_cast<const T *>(p)[i]);
}

// e^-|z|'s form of the logistic function: s = 1 / (1 + e^-z) and its
// derivative e / (1 + e)^2, e = e^-|z|, which never subtracts near numbers.
// One exp2 and one reciprocal, 1 ulp each.
__device__ __forceinline__ void logistic(float z, float &s, float &d) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(z) * 1.4426950408889634f);
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    s = z >= 0.0f ? r : e * r;
    d = e * r * r;
}

constexpr float kTanhA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;

// Phi(-ax), ax = |x|: 2^q(t), q the degree-7 polynomial fitted to log2 Phi(-t)
// over [0, 6] for the least largest error of Phi, and 0 past 6 (Phi(-6) is
// 1e-9). Within 1.4e-7 of Phi everywhere (the fit 3.6e-8, Horner in fp32 and
// the exp2 the rest). common.h's gelu() has a fit of its own, weighted for
// x Phi alone: at x = 0 its Phi is 2.7e-6 off, which a derivative would show,
// and it keeps Phi(-6) past 6, which a product with a far x would.
__device__ __forceinline__ float phi_tail(float ax) {
    const float t = fminf(ax, 6.0f);
    float q = __builtin_fmaf(8.47016599e-06f, t, -5.39037901e-05f);
    q = __builtin_fmaf(q, t, -4.212356e-04f);
    q = __builtin_fmaf(q, t, 7.38927163e-03f);
    q = __builtin_fmaf(q, t, -5.26911095e-02f);
    q = __builtin_fmaf(q, t, -4.59153146e-01f);
    q = __builtin_fmaf(q, t, -1.15111089e+00f);
    q = __builtin_fmaf(q, t, -9.99999881e-01f);
    const float r = __builtin_amdgcn_exp2f(q);
    return ax > 6.0f ? 0.0f : r;
}

// The activation. gelu, gelu_tanh, silu and lrelu of slope 0 of minus infinity
// are their limit 0 (an infinity is kept out of a product with 0); NaN stays
// NaN.
__device__ __forceinline__ float act_fwd(int act, float slope, float z) {
    if (act == MXO_NONE) return z;
    if (act == MXO_LRELU) {
        const float c = slope == 0.0f && z == -__builtin_inff() ? -1.0f : z;
        return z >= 0.0f ? z : slope * c;
    }
    float v, d;
    if (act == MXO_GELU) {
        v = fmaxf(z, 0.0f) - fminf(fabsf(z), 6.0f) * phi_tail(fabsf(z));
    } else if (act == MXO_SIGMOID) {
        logistic(z, v, d);
    } else {
        const float c = fmaxf(z, -1e4f);
        const float u = act == MXO_SILU ? c : kTanhA * c * __builtin_fmaf(kTanhB * c, c, 1.0f);
        float s;
        logistic(u, s, d);
        v = c * s;
    }
    return z != z ? z : v;
}

template <int E>
__device__ __forceinline__ void act_fwd_n(int act, float slope, float *v) {
    // the choice once for all of them
#define OPS_ACT(which)                                                 \
    case which:                                                        \
        _Pragma("unroll") for (int e = 0; e < E; ++e) v[e] = act_fwd(which, slope, v[e]); \
        break;
    switch (act) {
        OPS_ACT(MXO_GELU)
        OPS_ACT(MXO_GELU_TANH)
        OPS_ACT(MXO_SILU)
        OPS_ACT(MXO_LRELU)
        OPS_ACT(MXO_SIGMOID)
        default: break;
    }
}

// Its derivative; at an infinity its limit, at NaN NaN (LeakyReLU: of a NaN
// the slope, as its comparison gives).
__device__ __forceinline__ float act_bwd(int act, float slope, float z) {
    if (act == MXO_NONE) return 1.0f;
    if (act == MXO_LRELU) return z >= 0.0f ? 1.0f : slope;
    float v, s, d;
    if (act == MXO_GELU) {
        // Phi(z) + z phi(z); past |z| = 13 the density's term is below 3e-36
        const float ax = fabsf(z), t = fminf(ax, 13.0f);
        const float p = phi_tail(ax), g = 0.3989422804014327f * __builtin_amdgcn_exp2f(t * t * -0.7213475204444817f);
        v = (z >= 0.0f ? 1.0f - p : p) + copysignf(t, z) * g;
    } else if (act == MXO_SIGMOID) {
        logistic(z, s, v);
    } else if (act == MXO_SILU) {
        const float c = fminf(fmaxf(z, -1e4f), 1e4f);
        logistic(c, s, d);
        v = __builtin_fmaf(c, d, s);
    } else {
        const float c = fminf(fmaxf(z, -1e4f), 1e4f);
        logistic(kTanhA * c * __builtin_fmaf(kTanhB * c, c, 1.0f), s, d);
        v = __builtin_fmaf(c * d, kTanhA * __builtin_fmaf(3.0f * kTanhB * c, c, 1.0f), s);
    }
    return z != z ? z : v;
}

// v[e] *= act'(z[e])
template <int E, typename Z>
__device__ __forceinline__ void act_bwd_n(int act, float slope, float *v, Z z) {
    switch (act) {
#undef OPS_ACT
#define OPS_ACT(which)                                                                     \
    case which:                                                                            \
        _Pragma("unroll") for (int e = 0; e < E; ++e) v[e] *= act_bwd(which, slope, z(e)); \
        break;
        OPS_ACT(MXO_GELU)
        OPS_ACT(MXO_GELU_TANH)
        OPS_ACT(MXO_SILU)
        OPS_ACT(MXO_LRELU)
        OPS_ACT(MXO_SIGMOID)
        default: break;
    }
#undef OPS_ACT
}

// Sum over the 64 lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}
