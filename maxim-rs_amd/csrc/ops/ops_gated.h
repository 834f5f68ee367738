// The gated Dense: z = x w^T + bias with w's rows (and z's features) in two
// halves (a | c), y = act(a) c, and the backward pass's dz.
//
// Forward it is a product whose epilogue needs two sums for a result. The
// tiles of ops_gemm.h take both: of a wave's rows of the weights' operand half
// are the gate's and half the values' of the same features (Tile's HALF), so
// its sums of a and of c lie in the same lanes, and neither z nor a second
// product goes through memory unless z is kept. The weights are B where
// features are contiguous in the results (PAIR_N), A in planar order (PAIR_M).
// As a product of twice the columns: 8192 x 2048 to 2 x 4096 bf16 225 us a call,
// with z (134 MB more) 229 to 242 by the card's clock (the product alone, of
// which all of z is stored, 222 to 227); 64 to 2 x 64 fp32 planes of 65536 with z,
// 67 MB, 18.4 us, 3.6 TB/s.
#pragma once

#include "ops_gemm_big.h"

// What E results of row m need from memory: one bias of each half where it
// runs along the rows.
template <typename T>
struct GatedBias {
    float a, c;
};
template <typename T>
__device__ __forceinline__ GatedBias<T> gated_bias_row(const OpsGemmArgs &g, int64_t m) {
    if (!g.bias || !g.bias_rows || m >= g.m) return {0.0f, 0.0f};
    return {param<T>(g.bias, m, g.bias_f32), param<T>(g.bias, m + g.m, g.bias_f32)};
}
// The biases of columns n on, zeros where they run along the rows.
template <typename T, int E>
__device__ __forceinline__ void gated_bias_cols(const OpsGemmArgs &g, int64_t n, float *a, float *c) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool in = g.bias && !g.bias_rows && n + e < g.n;
        a[e] = in ? param<T>(g.bias, n + e, g.bias_f32) : 0.0f;
        c[e] = in ? param<T>(g.bias, n + e + g.n, g.bias_f32) : 0.0f;
    }
}

// y and z for E consecutive n of row m from the sums of both halves. The sums,
// the activation and the product are fp32, each store rounds once.
template <typename T, int E, int PAIR>
__device__ __forceinline__ void gated_finish(const OpsGemmArgs &g, int64_t m, int64_t n, float *a, float *c) {
    if (m >= g.m || n >= g.n) return;
    const int64_t have = g.n - n;
    Vec<T, E> o;
    if (g.z) {
        T *z = static_cast<T *>(g.z) + m * g.ldz + n;
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(a[e]);
        store_out<T, E>(z, o, have);
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(c[e]);
        store_out<T, E>(z + (PAIR == PAIR_N ? (int64_t)g.n : g.m * g.ldz), o, have);
    }
    act_fwd_n<E>(g.act, g.slope, a);
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(a[e] * c[e]);
    store_out<T, E>(static_cast<T *>(g.c) + m * g.ldc + n, o, have);
}

// Where split s's partial sums of row m, column n of a half lie: [splits][m][2 n]
// or [splits][2 m][n].
template <int PAIR>
__device__ __forceinline__ float *gated_part(const OpsGemmArgs &g, int s, int64_t m, int64_t n) {
    return g.part + ((int64_t)s * g.m * (PAIR == PAIR_M ? 2 : 1) + m) * ((int64_t)g.n * (PAIR == PAIR_N ? 2 : 1)) + n;
}
template <int PAIR>
__device__ __forceinline__ int64_t gated_part_half(const OpsGemmArgs &g) {
    return PAIR == PAIR_N ? (int64_t)g.n : (int64_t)g.m * g.n;
}

// A wave's FM x FN blocks of 16 x 16 sums, which are half as many results from
// (m0, n0) on: gemm_write's way through LDS, 32 rows at a time with both halves
// in a row (PAIR_N), or 16 rows of each half (PAIR_M).
template <typename T, int FM, int FN, int PAIR>
__device__ __forceinline__ void gated_write(const OpsGemmArgs &g, int64_t m0, int64_t n0, int s, int l, char *at,
                                            const f32x4 (&acc)[FM][FN]) {
    constexpr int E = 16 / sizeof(T), LD = FN * 16 + 4;
    constexpr bool ONE = PAIR == PAIR_N && FN > 4;  // a block of rows at a time, not two
    constexpr int COLS = PAIR == PAIR_N ? FN * 8 : FN * 16, TALL = PAIR == PAIR_N && !ONE ? 32 : 16;
    constexpr int LANES = COLS / E, ROWS = 64 / LANES < TALL ? 64 / LANES : TALL, STEPS = TALL / ROWS;
    constexpr int OTHER = PAIR == PAIR_N ? COLS : 16 * LD;  // a value's sum from its gate's
    static_assert(FM % 2 == 0 && FN % 2 == 0 && LANES * ROWS == 64, "");
    float *own = reinterpret_cast<float *>(at);
    const int lr = l / LANES, lc = l % LANES * E;
    const int64_t n = n0 + lc;
    float ba[E], bc[E];
    const bool whole = g.splits == 1;
    if (whole) gated_bias_cols<T, E>(g, n, ba, bc);
#pragma unroll 1
    for (int h = 0; h < (ONE ? FM : FM / 2); ++h) {
        const int64_t m = m0 + h * TALL + lr;
        GatedBias<T> row[STEPS];
        if (PAIR == PAIR_M && whole) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k) row[k] = gated_bias_row<T>(g, m + k * ROWS);
        }
#pragma unroll
        for (int i = 0; i < (ONE ? FM : FM / 2); ++i)
            if (i == h) {
                if (ONE) put_rows(own, l, acc, i, -1);
                else put_rows(own, l, acc, PAIR == PAIR_N ? 2 * i : i, PAIR == PAIR_N ? 2 * i + 1 : i + FM / 2);
                own_path(i);
            }
        wave_fence();
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            float a[E], c[E];
            const float *p = own + (k * ROWS + lr) * LD + lc;
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                *reinterpret_cast<f32x4 *>(a + e) = *reinterpret_cast<const f32x4 *>(p + e);
                *reinterpret_cast<f32x4 *>(c + e) = *reinterpret_cast<const f32x4 *>(p + OTHER + e);
            }
            if (whole) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    a[e] += PAIR == PAIR_M ? row[k].a : ba[e];
                    c[e] += PAIR == PAIR_M ? row[k].c : bc[e];
                }
                gated_finish<T, E, PAIR>(g, m + k * ROWS, n, a, c);
            } else if (m + k * ROWS < g.m && n < g.n) {
                float *o = gated_part<PAIR>(g, s, m + k * ROWS, n);
                store_upto<float, E>(o, __builtin_bit_cast(Vec<float, E>, a), g.n - n);
                store_upto<float, E>(o + gated_part_half<PAIR>(g), __builtin_bit_cast(Vec<float, E>, c), g.n - n);
            }
        }
        wave_fence();
    }
}

// The splits' sums of both halves added in a fixed order, then the epilogue:
// WAYS threads to four results, each every WAYS-th split, joined through LDS.
template <typename T, int WAYS, int PAIR>
__device__ __forceinline__ void gated_join(const OpsGemmArgs &g) {
    constexpr int Q = 256 / WAYS;
    __shared__ f32x4 sh[2][WAYS > 1 ? 256 : 1];
    const int64_t quads = ((int64_t)g.n + 3) / 4, total = quads * g.m, half = gated_part_half<PAIR>(g);
    const int64_t plane = 2 * (int64_t)g.m * g.n;
    const int q = threadIdx.x % Q, way = threadIdx.x / Q;
    for (int64_t i0 = (int64_t)blockIdx.x * Q; i0 < total; i0 += (int64_t)gridDim.x * Q) {
        const int64_t i = i0 + q, m = i / quads, n = (i - m * quads) * 4;
        f32x4 a = {0, 0, 0, 0}, c = a;
        if (i < total) {
            const float *p = gated_part<PAIR>(g, 0, m, n);
#pragma unroll 4
            for (int s = way; s < g.splits; s += WAYS) {
                const Vec<float, 4> va = load_upto<float, 4>(p + s * plane, g.n - n);
                const Vec<float, 4> vc = load_upto<float, 4>(p + s * plane + half, g.n - n);
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] += va.v[e], c[e] += vc.v[e];
            }
        }
        if constexpr (WAYS > 1) {
            __syncthreads();
            sh[0][threadIdx.x] = a;
            sh[1][threadIdx.x] = c;
            __syncthreads();
            if (way) continue;
#pragma unroll
            for (int k = 1; k < WAYS; ++k) a += sh[0][k * Q + q], c += sh[1][k * Q + q];
        }
        if (i >= total) continue;
        float ra[4], rc[4], ba[4], bc[4];
        gated_bias_cols<T, 4>(g, n, ba, bc);
        const GatedBias<T> row = gated_bias_row<T>(g, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) ra[e] = a[e] + ba[e] + row.a, rc[e] = c[e] + bc[e] + row.c;
        gated_finish<T, 4, PAIR>(g, m, n, ra, rc);
    }
}

// Up to 16 rows: ops_skinny.h's way, the block's 16 features of both halves at
// once, each weight read once (1 x 2048 to 2 x 8192 bf16, 67 MB: 15.1 us, 4.4
// TB/s).
template <typename T>
__device__ __forceinline__ void gated_skinny(const OpsGemmArgs &g) {
    constexpr int E = 16 / sizeof(T), STEP = 4 * E, W = 8, AHEAD = 4;
    typedef typename Mma<T>::Frag Frag;
    __shared__ f32x4 sums[2][W][64];
    const int t = threadIdx.x, l = t & 63, w = t >> 6, r = l & 15, q = l >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int each = (g.k + W * STEP - 1) / (W * STEP) * STEP, kbeg = w * each + q * E, kend = min(g.k, (w + 1) * each);
    const T *b = static_cast<const T *>(g.b) + min(n0 + r, (int64_t)g.n - 1) * g.ldb;
    const T *c = b + (int64_t)g.n * g.ldb;
    const T *a = static_cast<const T *>(g.a) + (int64_t)min(r, g.m - 1) * g.lda;
    f32x4 gate = {0, 0, 0, 0}, value = gate;
    const int steps = each / STEP, whole = max(0, (kend - w * each)) / STEP;
    auto go = [&](const Vec<T, E> &fb, const Vec<T, E> &fc, const Vec<T, E> &fa) {
        gate = Mma<T>::go(__builtin_bit_cast(Frag, fb), __builtin_bit_cast(Frag, fa), gate);
        value = Mma<T>::go(__builtin_bit_cast(Frag, fc), __builtin_bit_cast(Frag, fa), value);
    };
    int s = 0;
    for (; s + AHEAD <= whole; s += AHEAD) {
        Vec<T, E> fb[AHEAD], fc[AHEAD], fa[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int k = kbeg + (s + j) * STEP;
            fb[j] = load_n<T, E>(b + k);
            fc[j] = load_n<T, E>(c + k);
            fa[j] = load_n<T, E>(a + k);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) go(fb[j], fc[j], fa[j]);
    }
    for (; s < steps; ++s) {
        const int k = kbeg + s * STEP;
        go(load_upto<T, E>(b + k, kend - k), load_upto<T, E>(c + k, kend - k), load_upto<T, E>(a + k, kend - k));
    }
    sums[0][w][l] = gate;
    sums[1][w][l] = value;
    __syncthreads();
    if (t >= 64) return;
    gate = sums[0][0][l], value = sums[1][0][l];
#pragma unroll
    for (int k = 1; k < W; ++k) gate += sums[0][k][l], value += sums[1][k][l];
    // lane l: row l % 16, columns 4 (l / 16) + 0..3
    const int64_t m = r, n = n0 + q * 4;
    float ra[4], rc[4], ba[4], bc[4];
    gated_bias_cols<T, 4>(g, n, ba, bc);
    const GatedBias<T> row = gated_bias_row<T>(g, m);
#pragma unroll
    for (int e = 0; e < 4; ++e) ra[e] = gate[e] + ba[e] + row.a, rc[e] = value[e] + bc[e] + row.c;
    gated_finish<T, 4, PAIR_N>(g, m, n, ra, rc);
}

// dz = (dy c act'(a) | dy act(a)) and the bias's partial sums, one pass over dy
// and z. Stored rounded to the operands' type, as the products' matrix cores
// take it (ops_rows.h has what that costs); the bias's sums take it before. Bound
// by memory: 4096 x 2 x 2048 bf16, 84 MB, 15.5 us; 64 fp32 planes of 71680, 92 MB,
// 16 us.
//
// act(z) and act'(z) as act_fwd and act_bwd have them, with what they share
// formed once: an exponential and a reciprocal instead of two (the planar pass
// of 64 bf16 features, silu, 71680 positions: 14.4 us, so 13.1).
__device__ __forceinline__ void act_both(int act, float slope, float z, float &f, float &d) {
    if (act == MXO_GELU) {
        const float ax = fabsf(z), t = fminf(ax, 13.0f), p = phi_tail(ax);
        f = fmaxf(z, 0.0f) - fminf(ax, 6.0f) * p;
        d = (z >= 0.0f ? 1.0f - p : p) +
            copysignf(t, z) * (0.3989422804014327f * __builtin_amdgcn_exp2f(t * t * -0.7213475204444817f));
    } else if (act == MXO_SIGMOID) {
        logistic(z, f, d);
    } else if (act == MXO_SILU || act == MXO_GELU_TANH) {
        const float c = fminf(fmaxf(z, -1e4f), 1e4f), q = kTanhB * c * c;
        float s, e;
        logistic(act == MXO_SILU ? c : kTanhA * c * (q + 1.0f), s, e);
        f = fmaxf(z, -1e4f) * s;
        d = __builtin_fmaf(act == MXO_SILU ? c : c * kTanhA * __builtin_fmaf(3.0f, q, 1.0f), e, s);
    } else {
        f = act_fwd(act, slope, z);
        d = act_bwd(act, slope, z);
        return;
    }
    f = z != z ? z : f;
    d = z != z ? z : d;
}

// v: dy in, da out; u: a in, dc out.
template <int E>
__device__ __forceinline__ void gated_dz_n(int act, float slope, float *v, float *u, const float *c) {
#define OPS_DZ(which)                                                  \
    case which:                                                        \
        _Pragma("unroll") for (int e = 0; e < E; ++e) {                \
            float f, d;                                                \
            act_both(which, slope, u[e], f, d);                        \
            u[e] = v[e] * f, v[e] = v[e] * c[e] * d;                   \
        }                                                              \
        break;
    switch (act) {
        OPS_DZ(MXO_NONE)
        OPS_DZ(MXO_GELU)
        OPS_DZ(MXO_GELU_TANH)
        OPS_DZ(MXO_SILU)
        OPS_DZ(MXO_LRELU)
        OPS_DZ(MXO_SIGMOID)
        default: break;
    }
#undef OPS_DZ
}

__device__ __forceinline__ void store_sum(void *out, int dtype, int64_t i, float v) {
    if (dtype == MXO_F32) static_cast<float *>(out)[i] = v;
    else if (dtype == MXO_F16) static_cast<f16 *>(out)[i] = from_f<f16>(v);
    else static_cast<bf16 *>(out)[i] = from_f<bf16>(v);
}
// A part's sum of feature i of 2 cols.
__device__ __forceinline__ void keep_sum(const OpsGatedDzArgs &g, int64_t part, int64_t i, float v) {
    if (g.db) store_sum(g.db, g.db_type, i, v);
    else g.d.part[2 * part * g.d.cols + i] = v;
}

// dz in fp16. A product of three values leaves fp16's range where the gradients
// it leads to do not: past 65504 it would be infinite, and below 2^-14 it loses
// bits. So the pass keeps each block's largest finite |dz| (`top`), and a second
// launch of it, from the largest of all: 1 to 65520, or nothing: dz is right as it
// is, and the blocks leave; else they form dz again, times the power of two that
// takes the largest into [2^14, 2^15), which the products' sums are divided by.
// An element is off by half a step of its own, or by 2^-25 as it is and 2^-39 of
// the largest where it was scaled. (One scale for all: a row's own would do for dx, whose sums stay in a row, but not for dw.
// Scaling always would take a pass over dy and z before this one.) A backward pass
// of 4096 x 1024 to 2 x 2048 takes 99 us without any of this, 105 with dz in range
// (the magnitudes 1, the launch that leaves 3 to 4) and 113 with dz out of it; 64 to
// 2 x 64 planes of 71680 30, 34 and 44.
template <typename T>
constexpr bool kScaled = __is_same(T, f16);
// The largest of 256 threads' values, in all of them.
__device__ __forceinline__ float block_top(float v) {
    __shared__ float at[4];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(at[0], at[1]), fmaxf(at[2], at[3]));
}
// The larger of `top` and the finite magnitudes of v and u (NaN drops out of a
// maximum by itself).
template <int E>
__device__ __forceinline__ float top_of(float top, const float *v, const float *u) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(fmaxf(m, fabsf(v[e])), fabsf(u[e]));
    if (m == __builtin_inff()) {
        m = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float a = fabsf(v[e]), b = fabsf(u[e]);
            m = fmaxf(fmaxf(m, a < __builtin_inff() ? a : 0.0f), b < __builtin_inff() ? b : 0.0f);
        }
    }
    return fmaxf(top, m);
}
__device__ __forceinline__ void keep_top(const OpsGatedDzArgs &g, float v) {
    if (!g.top) return;
    v = block_top(v);
    if (threadIdx.x == 0) g.top[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = v;
}
// What this launch's dz is multiplied by; 0: there is nothing to do. Many blocks'
// magnitudes are brought to one by a launch of their own (MXO_DZ_TOPS), not by
// every block.
__device__ __forceinline__ float dz_scale(const OpsGatedDzArgs &g) {
    if (g.pass == MXO_DZ) return 1.0f;
    float v = 0.0f;
#pragma unroll 8
    for (int i = threadIdx.x; i < g.ntop; i += 256) v = fmaxf(v, g.top[i]);
    v = block_top(v);
    if (g.pass == MXO_DZ_TOPS) {
        if (threadIdx.x == 0) g.top[g.ntop] = v;
        return 0.0f;
    }
    const bool fits = v == 0.0f || (v >= 1.0f && v < 65520.0f);
    // (it multiplies dy, exactly, and 2^60 at most keeps what follows finite)
    const int e = fits ? 0 : min(14 + 127 - (int)(__builtin_bit_cast(uint32_t, v) >> 23), 60);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *g.back = __builtin_bit_cast(float, (127 - e) << 23);
    return fits ? 0.0f : __builtin_bit_cast(float, (127 + e) << 23);
}

// Rows with contiguous features: 64 x E features by a run of rows a block, a
// wave a row at a time.
template <typename T, bool WHOLE>
__device__ __forceinline__ void gated_dz_rows(const OpsGatedDzArgs &g, float (*sh)[2][64 * 16 / sizeof(T)]) {
    const OpsDzArgs &a = g.d;
    constexpr int E = 16 / sizeof(T);
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + l) * E, p = blockIdx.y, have = a.cols - c;
    // (the second launch's blocks take longer runs)
    const int nparts = kScaled<T> ? (int)gridDim.y : a.nparts;
    const int64_t chunk = (a.rows + nparts - 1) / nparts, end = min(a.rows, (p + 1) * chunk);
    float scale = 1.0f, top = 0.0f;
    if constexpr (kScaled<T>)
        if ((scale = dz_scale(g)) == 0.0f) return;
    float sa[E], sc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sa[e] = sc[e] = 0.0f;
    if (have > 0)
        for (int64_t r = p * chunk + w; r < end; r += 4) {
            const T *dy = static_cast<const T *>(a.dy) + r * a.dyrs + c, *z = static_cast<const T *>(a.z) + r * a.zrs + c;
            // a lane without features has left already
            const int64_t rest = a.rows - 1 - r, last = a.cols - E - c;
            const u32x4 vd = load_in<T, E, WHOLE>(dy, dy, dy + rest * a.dyrs + last, have);
            const u32x4 vz = load_in<T, E, WHOLE>(z, z, z + rest * a.zrs + last, have);
            const u32x4 vc = load_in<T, E, WHOLE>(z + a.cols, z + a.cols, z + a.cols + rest * a.zrs + last, have);
            float v[E], u[E], m[E];
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = elem<T>(vd, e), u[e] = elem<T>(vz, e), m[e] = elem<T>(vc, e);
            if constexpr (kScaled<T>) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] *= scale;
            }
            gated_dz_n<E>(a.act, a.slope, v, u, m);
            if constexpr (kScaled<T>) top = top_of<E>(top, v, u);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                // features past the last are not there to be summed or stored
                sa[e] += v[e], sc[e] += u[e];
                o.v[e] = from_f<T>(v[e]);
            }
            if (a.dz) {
                T *dz = static_cast<T *>(a.dz) + r * a.drs + c;
                store_in<T, E, WHOLE>(dz, o, have);
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(u[e]);
                store_in<T, E, WHOLE>(dz + a.cols, o, have);
                // the products' loads take lines of whole vectors, zeros at their ends
                if (!WHOLE && have <= E)
                    for (int64_t k = 2 * a.cols - c; k < a.drs - c; ++k) dz[k] = (T)0.0f;
            }
        }
    if constexpr (kScaled<T>) {
        if (g.pass != MXO_DZ) return;  // the sums are there
        keep_top(g, top);
    }
    if (!a.part && !g.db) return;
#pragma unroll
    for (int e = 0; e < E; ++e) sh[w][0][l * E + e] = sa[e], sh[w][1][l * E + e] = sc[e];
    __syncthreads();
    for (int k = threadIdx.x; k < 128 * E; k += 256) {
        const int h = k >= 64 * E, i = k - h * 64 * E;
        const int64_t col = (int64_t)blockIdx.x * 64 * E + i;
        if (col < a.cols)
            keep_sum(g, p, h * a.cols + col, (sh[0][h][i] + sh[1][h][i]) + (sh[2][h][i] + sh[3][h][i]));
    }
}
// Planar order: one feature by a run of positions a block.
template <typename T>
__device__ __forceinline__ void gated_dz_planar(const OpsGatedDzArgs &g) {
    const OpsDzArgs &a = g.d;
    constexpr int E = 16 / sizeof(T);
    __shared__ float sh[2][4];
    const int64_t c = blockIdx.x, p = blockIdx.y;
    const int nparts = kScaled<T> ? (int)gridDim.y : a.nparts;
    const int64_t chunk = ((a.rows + nparts - 1) / nparts + E - 1) / E * E, end = min(a.rows, (p + 1) * chunk);
    const T *dy = static_cast<const T *>(a.dy) + c * a.dycs, *z = static_cast<const T *>(a.z) + c * a.zcs;
    T *dz = static_cast<T *>(a.dz) + c * a.dcs;
    float sa = 0.0f, sc = 0.0f, scale = 1.0f, top = 0.0f;
    if constexpr (kScaled<T>)
        if ((scale = dz_scale(g)) == 0.0f) return;
    for (int64_t r = p * chunk + threadIdx.x * E; r < end; r += 256 * E) {
        const Vec<T, E> vd = load_upto<T, E>(dy + r, end - r), vz = load_upto<T, E>(z + r, end - r);
        const Vec<T, E> vc = load_upto<T, E>(z + a.cols * a.zcs + r, end - r);
        float v[E], u[E], m[E];
        Vec<T, E> oa, oc;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = to_f<T>(vd.v[e]), u[e] = to_f<T>(vz.v[e]), m[e] = to_f<T>(vc.v[e]);
        if constexpr (kScaled<T>) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] *= scale;
        }
        gated_dz_n<E>(a.act, a.slope, v, u, m);
        // (past the end dy is 0, and so is dz)
        if constexpr (kScaled<T>) top = top_of<E>(top, v, u);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (r + e < end) sa += v[e], sc += u[e];
            oa.v[e] = from_f<T>(v[e]), oc.v[e] = from_f<T>(u[e]);
        }
        // lines of dz are whole vectors, their ends zeros (a run is whole vectors)
        if (a.dz) {
            store_n<T, E>(dz + r, oa);
            store_n<T, E>(dz + a.cols * a.dcs + r, oc);
        }
    }
    if constexpr (kScaled<T>) {
        if (g.pass != MXO_DZ) return;
        keep_top(g, top);
    }
    if (!a.part && !g.db) return;
    sa = wave_sum(sa), sc = wave_sum(sc);
    if ((threadIdx.x & 63) == 0) sh[0][threadIdx.x >> 6] = sa, sh[1][threadIdx.x >> 6] = sc;
    __syncthreads();
    if (threadIdx.x < 2) {
        const float *s = sh[threadIdx.x];
        keep_sum(g, p, threadIdx.x * a.cols + c, (s[0] + s[1]) + (s[2] + s[3]));
    }
}

// The joins of dw's splits and of the bias's partial sums. Few results and many
// parts: 16 threads to four of dw's, 64 to a bias's, 16 parts in turn each at
// most in flight, added in a fixed order. (128 x 64 results of 249 parts and 128
// of 35, fp32: 12 us as two launches of their own, so 5.8.)
template <typename T>
__device__ __forceinline__ void grad_join(const OpsGradJoinArgs &a) {
    __shared__ f32x4 sh[256];
    const int t = threadIdx.x;
    if ((int)blockIdx.x >= a.first) {
        // four columns a block, 64 threads down the parts
        float *s = reinterpret_cast<float *>(sh);
        const int l = t & 3, w = t >> 2;
        const int64_t c = ((int64_t)blockIdx.x - a.first) * 4 + l;
        float v = 0.0f;
        if (c < a.n) {
#pragma unroll 4
            for (int i = w; i < a.nparts; i += 64) v += a.part[(int64_t)i * a.n + c];
        }
        s[t] = v;
#pragma unroll
        for (int half = 32; half >= 1; half >>= 1) {
            __syncthreads();
            if (w < half) s[t] += s[t + half * 4];
        }
        if (w == 0 && c < a.n) store_sum(a.out, a.dtype, c, s[t]);
        return;
    }
    const OpsGemmArgs &g = a.g;
    const int64_t quads = ((int64_t)g.n + 3) / 4, total = quads * g.m, plane = (int64_t)g.m * g.n;
    const int q = t & 15, way = t >> 4;
    const float back = back_of<T>(g);
    for (int64_t i0 = (int64_t)blockIdx.x * 16; i0 < total; i0 += (int64_t)a.first * 16) {
        const int64_t i = i0 + q, m = i / quads, n = (i - m * quads) * 4;
        f32x4 v = {0, 0, 0, 0};
        if (i < total) {
            const float *p = g.part + m * g.n + n;
#pragma unroll 4
            for (int s = way; s < g.splits; s += 16) {
                const Vec<float, 4> o = load_upto<float, 4>(p + s * plane, g.n - n);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += o.v[e];
            }
        }
        __syncthreads();
        sh[t] = v;
        __syncthreads();
        if (way || i >= total) continue;
#pragma unroll
        for (int k = 1; k < 16; ++k) v += sh[k * 16 + q];
        float r[4] = {v[0], v[1], v[2], v[3]};
        scale_back<T, 4>(r, back);
        Vec<T, 4> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] = from_f<T>(r[e]);
        store_upto<T, 4>(static_cast<T *>(g.c) + m * g.ldc + n, o, g.n - n);
    }
}

#define OPS_GATED1(name, T, B, WM, WN, axis, PAIR, tag, AK, BK)                                                  \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxg_gemm_##axis##_##name##_##B##x##B##_##tag(     \
        OpsGemmArgs g) {                                                                                         \
        __shared__ __align__(128) char lds[4 * B * 128];                                                         \
        gemm_tile<T, B, B, WM, WN, AK, BK, PAIR>(g, lds);                                                        \
    }
#define OPS_GATED_D2(name, T, B, WM, WN, axis, PAIR, tag, AK, BK)                                                \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxg_gemm_##axis##_##name##_##B##x##B##_##tag##_d2( \
        OpsGemmArgs g) {                                                                                         \
        OPS_STAGE(0, B, B)                                                                                       \
        OPS_STAGE(1, B, B)                                                                                       \
        const Stage st[2] = {{a0, b0}, {a1, b1}};                                                                \
        gemm_direct<T, B, B, WM, WN, AK, BK, 2, PAIR>(g, st);                                                    \
    }
#define OPS_GATED_D4(name, T, B, WM, WN, axis, PAIR, tag, AK, BK)                                                \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxg_gemm_##axis##_##name##_##B##x##B##_##tag##_d4( \
        OpsGemmArgs g) {                                                                                         \
        OPS_STAGE(0, B, B)                                                                                       \
        OPS_STAGE(1, B, B)                                                                                       \
        OPS_STAGE(2, B, B)                                                                                       \
        OPS_STAGE(3, B, B)                                                                                       \
        const Stage st[4] = {{a0, b0}, {a1, b1}, {a2, b2}, {a3, b3}};                                            \
        gemm_direct<T, B, B, WM, WN, AK, BK, 4, PAIR>(g, st);                                                    \
    }
// x has the results' order: rows along k with w either way (PAIR_N), or planes
#define OPS_GATED_ROWS(KIND, name, T, B, WM, WN)                       \
    KIND(name, T, B, WM, WN, n, PAIR_N, kk, true, true)                \
    KIND(name, T, B, WM, WN, n, PAIR_N, km, true, false)
#define OPS_GATED_PLANES(KIND, name, T, B, WM, WN)                     \
    KIND(name, T, B, WM, WN, m, PAIR_M, km, true, false)               \
    KIND(name, T, B, WM, WN, m, PAIR_M, mm, false, false)
#define OPS_GATED_ALL(KIND, name, T, B, WM, WN)                        \
    OPS_GATED_ROWS(KIND, name, T, B, WM, WN)                           \
    OPS_GATED_PLANES(KIND, name, T, B, WM, WN)
#define OPS_GATED_JOIN(name, T, axis, PAIR)                                                                              \
    extern "C" __global__ __launch_bounds__(256) void mxg_join_##axis##_##name(OpsGemmArgs g) { gated_join<T, 1, PAIR>(g); } \
    extern "C" __global__ __launch_bounds__(256) void mxg_join8_##axis##_##name(OpsGemmArgs g) { gated_join<T, 8, PAIR>(g); }
#define OPS_GATED_TYPE(name, T)                                                                                          \
    OPS_GATED_ALL(OPS_GATED1, name, T, 64, 2, 2)                                                                         \
    OPS_GATED_JOIN(name, T, n, PAIR_N)                                                                                   \
    OPS_GATED_JOIN(name, T, m, PAIR_M)                                                                                   \
    extern "C" __global__ __launch_bounds__(512) void mxg_skinny_##name(OpsGemmArgs g) { gated_skinny<T>(g); }           \
    extern "C" __global__ __launch_bounds__(256) void mxg_grad_join_##name(OpsGradJoinArgs a) { grad_join<T>(a); }        \
    extern "C" __global__ __launch_bounds__(256) void mxg_dz_rows_##name(OpsGatedDzArgs a) {                                  \
        __shared__ float sh[4][2][64 * 16 / sizeof(T)];                                                                  \
        if (a.d.cols % (16 / sizeof(T)) == 0) gated_dz_rows<T, true>(a, sh);                                               \
        else gated_dz_rows<T, false>(a, sh);                                                                             \
    }                                                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void mxg_dz_planar_##name(OpsGatedDzArgs a) { gated_dz_planar<T>(a); }

OPS_GATED_TYPE(bf16, bf16)
OPS_GATED_TYPE(f16, f16)
OPS_GATED_TYPE(f32, float)
// 256 x 256: waves whose results are 64 wide, whole lines of y and z (with half
// lines 8192 x 2048 to 2 x 4096 with z took 256 us, so 231); with w contiguous
// along its rows they do not fit the registers
OPS_GATED_D2(bf16, bf16, 256, 4, 2, n, PAIR_N, kk, true, true)
OPS_GATED_D2(f16, f16, 256, 4, 2, n, PAIR_N, kk, true, true)
OPS_GATED_D2(bf16, bf16, 256, 2, 4, n, PAIR_N, km, true, false)
OPS_GATED_D2(f16, f16, 256, 2, 4, n, PAIR_N, km, true, false)
OPS_GATED_PLANES(OPS_GATED_D2, bf16, bf16, 256, 2, 4)
OPS_GATED_PLANES(OPS_GATED_D2, f16, f16, 256, 2, 4)
OPS_GATED_ALL(OPS_GATED_D2, bf16, bf16, 128, 2, 2)
OPS_GATED_ALL(OPS_GATED_D2, f16, f16, 128, 2, 2)
OPS_GATED_ALL(OPS_GATED_D4, bf16, bf16, 128, 2, 2)
OPS_GATED_ALL(OPS_GATED_D4, f16, f16, 128, 2, 2)
OPS_GATED_ALL(OPS_GATED_D4, bf16, bf16, 64, 2, 2)
OPS_GATED_ALL(OPS_GATED_D4, f16, f16, 64, 2, 2)
OPS_GATED_ALL(OPS_GATED_D2, f32, float, 128, 2, 2)
OPS_GATED_ALL(OPS_GATED_D4, f32, float, 64, 2, 2)
OPS_GATED_ALL(OPS_GATED_D2, f32, float, 64, 2, 2)
