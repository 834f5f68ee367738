// LayerNorm, its backward pass and the activation's derivative with the
// bias's gradient: passes over [rows][cols] activations of either order.
//
// All of them are bound by memory: a row (or, in planar order, a column of 64
// positions) is read once into registers, reduced there, and written from
// there. The gradients of the parameters are sums over all rows: each block
// keeps its own in registers over the rows it walks and writes one partial
// sum, and mxo_join_parts adds those in their order, so the bits do not depend
// on which block ran first.
#pragma once

#include "ops_common.h"

// Sum over groups of L consecutive lanes, in every lane.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// Two sums over the LPR threads of a row's group, in every thread. Groups of
// a wave or less need no barrier; larger ones leave their waves' sums in `at`
// ([2 buffers][2][waves of the block], `turn` choosing the buffer, so that
// one barrier a call is enough: a buffer is written again two calls on).
template <int LPR, int BT>
__device__ __forceinline__ void row_sum2(float &a, float &b, float *at, int turn) {
    a = lanes_sum<(LPR < 64 ? LPR : 64)>(a);
    b = lanes_sum<(LPR < 64 ? LPR : 64)>(b);
    if constexpr (LPR > 64) {
        constexpr int W = BT / 64, GW = LPR / 64;
        const int w = threadIdx.x >> 6, g0 = w / GW * GW;
        float *buf = at + (turn & 1) * 2 * W;
        if ((threadIdx.x & 63) == 0) buf[w] = a, buf[W + w] = b;
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < GW; ++i) a += buf[g0 + i], b += buf[W + g0 + i];
    }
}

// LayerNorm of rows with contiguous columns: LPR threads a row, NV vectors of
// 16 bytes a thread, so a row of up to LPR * NV * 16 bytes stays in
// registers between the mean, the variance about it and the result. The
// parameters are read once a block, which walks over rows.
template <typename T, int LPR, int NV, int BT>
__device__ __forceinline__ void ln_rows(const OpsLnArgs &a) {
    constexpr int E = 16 / sizeof(T), RPB = BT / LPR;
    __shared__ float at[4 * (BT / 64)];
    const int li = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const float n = (float)a.cols;
    float sc[NV][E], bi[NV][E];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = (int64_t)(j * LPR + li) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sc[j][e] = c + e < a.cols ? param<T>(a.scale, c + e, a.param_f32) : 0.0f;
            bi[j][e] = a.bias && c + e < a.cols ? param<T>(a.bias, c + e, a.param_f32) : 0.0f;
        }
    }
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + grp;
        const bool on = r < a.rows;
        const T *x = static_cast<const T *>(a.x) + (on ? r : 0) * a.xrs;
        Vec<T, E> v[NV];
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(j * LPR + li) * E;
            v[j] = load_upto<T, E>(x + c, on ? a.cols - c : 0);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) s += to_f<T>(v[j].v[e]);
        float zero = 0.0f;
        row_sum2<LPR, BT>(s, zero, at, turn++);
        // a division: the mean of equal values is that value
        const float mean = s / n;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = to_f<T>(v[j].v[e]) - mean;
                q += (int64_t)(j * LPR + li) * E + e < a.cols ? d * d : 0.0f;
            }
        zero = 0.0f;
        row_sum2<LPR, BT>(q, zero, at, turn++);
        const float rstd = 1.0f / sqrtf(q / n + a.eps);
        if (!on) continue;  // a whole group, behind its last barrier of the round
        T *y = static_cast<T *>(a.y) + r * a.yrs;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(j * LPR + li) * E;
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.v[e] = from_f<T>((to_f<T>(v[j].v[e]) - mean) * rstd * sc[j][e] + bi[j][e]);
            store_upto<T, E>(y + c, o, a.cols - c);
        }
        if (li == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// The backward pass in the same arrangement: dx from registers, the
// parameters' gradients summed in registers over the block's rows, then over
// its row groups in LDS.
template <typename T, int LPR, int NV, int BT>
__device__ __forceinline__ void ln_bwd_rows(const OpsLnBwdArgs &a) {
    constexpr int E = 16 / sizeof(T), RPB = BT / LPR;
    __shared__ float at[4 * (BT / 64)];
    __shared__ float sums[RPB > 1 ? BT * NV * E : 1];
    const int li = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const float n = (float)a.cols;
    float sc[NV][E], ds[NV][E], db[NV][E];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = (int64_t)(j * LPR + li) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sc[j][e] = c + e < a.cols ? param<T>(a.scale, c + e, a.param_f32) : 0.0f;
            ds[j][e] = db[j][e] = 0.0f;
        }
    }
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + grp;
        const bool on = r < a.rows;
        const int64_t rr = on ? r : 0;
        const float mean = a.mean[rr], rstd = on ? a.rstd[rr] : 0.0f;
        Vec<T, E> vx[NV], vd[NV], va[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (int64_t)(j * LPR + li) * E, have = on ? a.cols - c : 0;
            vx[j] = load_upto<T, E>(static_cast<const T *>(a.x) + rr * a.xrs + c, have);
            vd[j] = load_upto<T, E>(static_cast<const T *>(a.dy) + rr * a.dyrs + c, have);
            if (a.add) va[j] = load_upto<T, E>(static_cast<const T *>(a.add) + rr * a.ars + c, have);
        }
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                // past the row's end dy is 0, and so is what it adds (x's 0
                // makes a finite xh there: mean and rstd are the row's own)
                const float dy = to_f<T>(vd[j].v[e]);
                const bool in = (int64_t)(j * LPR + li) * E + e < a.cols;
                const float xh = in && on ? (to_f<T>(vx[j].v[e]) - mean) * rstd : 0.0f;
                const float g = dy * sc[j][e];
                s += g;
                q += g * xh;
                ds[j][e] += dy * xh;
                db[j][e] += dy;
            }
        if (a.dx) {
            row_sum2<LPR, BT>(s, q, at, turn++);
            s /= n;
            q /= n;
            if (on) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int64_t c = (int64_t)(j * LPR + li) * E;
                    Vec<T, E> o;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float xh = (to_f<T>(vx[j].v[e]) - mean) * rstd;
                        float v = rstd * (to_f<T>(vd[j].v[e]) * sc[j][e] - s - xh * q);
                        if (a.add) v += to_f<T>(va[j].v[e]);
                        o.v[e] = from_f<T>(v);
                    }
                    store_upto<T, E>(static_cast<T *>(a.dx) + r * a.dxrs + c, o, a.cols - c);
                }
            }
        }
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) sums[grp * (LPR * NV * E) + (j * LPR + li) * E + e] = which ? db[j][e] : ds[j][e];
            __syncthreads();
            for (int i = threadIdx.x; i < LPR * NV * E && i < a.cols; i += BT) {
                float s = 0.0f;
#pragma unroll 4
                for (int g = 0; g < RPB; ++g) s += sums[g * (LPR * NV * E) + i];
                part[which * a.cols + i] = s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (int64_t)(j * LPR + li) * E;
                Vec<float, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = which ? db[j][e] : ds[j][e];
                store_upto<float, E>(part + which * a.cols + c, o, a.cols - c);
            }
        }
    }
}

// Planar order: 64 positions a block (LP lanes of 16 bytes), S = BT / LP
// threads down the channels, CH channels a thread, all in registers. Sums
// over channels run over a thread's own, the wave's lanes and, through LDS,
// the block's waves.
template <typename T, int BT>
struct PlanarTile {
    static constexpr int E = 16 / sizeof(T), LP = 64 / E, S = BT / LP, W = BT / 64;
    // E sums a thread, one a position, over the block's channels
    static __device__ __forceinline__ void sum(float *v, float *at) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int o = LP; o < 64; o <<= 1) v[e] += __shfl_xor(v[e], o);
        __syncthreads();
        if (lane < LP)
#pragma unroll
            for (int e = 0; e < E; ++e) at[w * 64 + lane * E + e] = v[e];
        __syncthreads();
        const int p = (lane % LP) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) s += at[i * 64 + p + e];
            v[e] = s;
        }
    }
};

// LOOP: any number of channels, read again for each of the three passes.
template <typename T, int BT, int CH, bool LOOP>
__device__ __forceinline__ void ln_planar(const OpsLnArgs &a) {
    typedef PlanarTile<T, BT> P;
    constexpr int E = P::E, LP = P::LP, S = P::S;
    __shared__ float at[P::W * 64];
    const int pl = threadIdx.x % LP, sl = threadIdx.x / LP;
    const float n = (float)a.cols;
    const int rounds = LOOP ? (int)((a.cols + S * CH - 1) / (S * CH)) : 1;
    for (int64_t p0 = (int64_t)blockIdx.x * 64; p0 < a.rows; p0 += (int64_t)gridDim.x * 64) {
        const int64_t p = p0 + pl * E, have = a.rows - p;
        Vec<T, E> v[CH];
        auto fetch = [&](int round) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                v[j] = load_upto<T, E>(static_cast<const T *>(a.x) + c * a.xcs + p, c < a.cols ? have : 0);
            }
        };
        float s[E], q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] = q[e] = 0.0f;
        for (int round = 0; round < rounds; ++round) {
            fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] += to_f<T>(v[j].v[e]);
        }
        P::sum(s, at);
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] /= n;
        for (int round = 0; round < rounds; ++round) {
            if (LOOP) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const bool in = ((int64_t)round * CH + j) * S + sl < a.cols;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = to_f<T>(v[j].v[e]) - s[e];
                    q[e] += in ? d * d : 0.0f;
                }
            }
        }
        P::sum(q, at);
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = 1.0f / sqrtf(q[e] / n + a.eps);
        for (int round = 0; round < rounds; ++round) {
            if (LOOP) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                if (c >= a.cols) continue;
                const float sc = param<T>(a.scale, c, a.param_f32), bi = a.bias ? param<T>(a.bias, c, a.param_f32) : 0.0f;
                Vec<T, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = from_f<T>((to_f<T>(v[j].v[e]) - s[e]) * q[e] * sc + bi);
                store_upto<T, E>(static_cast<T *>(a.y) + c * a.ycs + p, o, have);
            }
        }
        if (sl == 0) {
            Vec<float, E> m, r;
#pragma unroll
            for (int e = 0; e < E; ++e) m.v[e] = s[e], r.v[e] = q[e];
            if (a.mean) store_upto<float, E>(a.mean + p, m, have);
            if (a.rstd) store_upto<float, E>(a.rstd + p, r, have);
        }
    }
}

template <typename T, int BT, int CH, bool LOOP>
__device__ __forceinline__ void ln_bwd_planar(const OpsLnBwdArgs &a) {
    typedef PlanarTile<T, BT> P;
    constexpr int E = P::E, LP = P::LP, S = P::S;
    __shared__ float at[P::W * 64];
    const int pl = threadIdx.x % LP, sl = threadIdx.x / LP;
    const float n = (float)a.cols;
    const int rounds = LOOP ? (int)((a.cols + S * CH - 1) / (S * CH)) : 1;
    float ds[CH], db[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) ds[j] = db[j] = 0.0f;
    for (int64_t p0 = (int64_t)blockIdx.x * 64; p0 < a.rows; p0 += (int64_t)gridDim.x * 64) {
        const int64_t p = p0 + pl * E, have = a.rows - p;
        Vec<T, E> vx[CH], vd[CH];
        auto fetch = [&](int round) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl, left = c < a.cols ? have : 0;
                vx[j] = load_upto<T, E>(static_cast<const T *>(a.x) + c * a.xcs + p, left);
                vd[j] = load_upto<T, E>(static_cast<const T *>(a.dy) + c * a.dycs + p, left);
            }
        };
        fetch(0);
        // past the last position rstd is 0, so what lies there adds nothing
        const Vec<float, E> m = load_upto<float, E>(a.mean + p, have), r = load_upto<float, E>(a.rstd + p, have);
        float s[E], q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] = q[e] = 0.0f;
        for (int round = 0; round < rounds; ++round) {
            if (round) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                const bool in = c < a.cols;
                const float sc = in ? param<T>(a.scale, c, a.param_f32) : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float dy = to_f<T>(vd[j].v[e]);
                    const float xh = in ? (to_f<T>(vx[j].v[e]) - m.v[e]) * r.v[e] : 0.0f;
                    s[e] += dy * sc;
                    q[e] += dy * sc * xh;
                    if (!LOOP) ds[j] += dy * xh, db[j] += dy;
                }
            }
        }
        if (!a.dx) continue;
        P::sum(s, at);
        P::sum(q, at);
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] /= n, q[e] /= n;
        for (int round = 0; round < rounds; ++round) {
            if (LOOP) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                if (c >= a.cols) continue;
                const float sc = param<T>(a.scale, c, a.param_f32);
                Vec<T, E> o, va;
                if (a.add) va = load_upto<T, E>(static_cast<const T *>(a.add) + c * a.acs + p, have);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float xh = (to_f<T>(vx[j].v[e]) - m.v[e]) * r.v[e];
                    float v = r.v[e] * (to_f<T>(vd[j].v[e]) * sc - s[e] - xh * q[e]);
                    if (a.add) v += to_f<T>(va.v[e]);
                    o.v[e] = from_f<T>(v);
                }
                store_upto<T, E>(static_cast<T *>(a.dx) + c * a.dxcs + p, o, have);
            }
        }
    }
    if (LOOP || !a.part) return;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const float s = lanes_sum<LP>(ds[j]), b = lanes_sum<LP>(db[j]);
        const int64_t c = (int64_t)j * S + sl;
        if (pl == 0 && c < a.cols) {
            a.part[((int64_t)blockIdx.x * 2) * a.cols + c] = s;
            a.part[((int64_t)blockIdx.x * 2 + 1) * a.cols + c] = b;
        }
    }
}

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

// Rows too long for registers: a block of 1024 threads a row, three passes
// over it, the later two from the caches.
template <typename T>
__device__ __forceinline__ void ln_long(const OpsLnArgs &a) {
    __shared__ float at[16];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.xrs;
        T *y = static_cast<T *>(a.y) + r * a.yrs;
        float s = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) s += to_f<T>(x[c]);
        const float mean = block_sum(s, at) / (float)a.cols;
        s = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float d = to_f<T>(x[c]) - mean;
            s += d * d;
        }
        const float rstd = 1.0f / sqrtf(block_sum(s, at) / (float)a.cols + a.eps);
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float d = (to_f<T>(x[c]) - mean) * rstd;
            const float b = a.bias ? param<T>(a.bias, c, a.param_f32) : 0.0f;
            y[c] = from_f<T>(d * param<T>(a.scale, c, a.param_f32) + b);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__device__ __forceinline__ void ln_bwd_long(const OpsLnBwdArgs &a) {
    __shared__ float at[16];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.xrs;
        const T *dy = static_cast<const T *>(a.dy) + r * a.dyrs;
        const T *add = a.add ? static_cast<const T *>(a.add) + r * a.ars : nullptr;
        T *dx = static_cast<T *>(a.dx) + r * a.dxrs;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s = 0.0f, q = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float gr = to_f<T>(dy[c]) * param<T>(a.scale, c, a.param_f32);
            s += gr;
            q += gr * ((to_f<T>(x[c]) - mean) * rstd);
        }
        s = block_sum(s, at) / (float)a.cols;
        q = block_sum(q, at) / (float)a.cols;
        for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
            const float gr = to_f<T>(dy[c]) * param<T>(a.scale, c, a.param_f32);
            const float xh = (to_f<T>(x[c]) - mean) * rstd;
            float v = rstd * (gr - s - xh * q);
            if (add) v += to_f<T>(add[c]);
            dx[c] = from_f<T>(v);
        }
    }
}

// The parameters' gradients alone, for rows too long for registers: 64 x E
// columns by a run of rows a block, four waves each a quarter of the rows; in
// planar order one channel by a run of positions a block.
template <typename T>
__device__ __forceinline__ void ln_param_rows(const OpsLnBwdArgs &a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float sh[2][4][64 * E];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + l) * E, p = blockIdx.y, have = a.cols - c;
    const int64_t chunk = (a.rows + a.nparts - 1) / a.nparts, end = min(a.rows, (p + 1) * chunk);
    float s[E], b[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = b[e] = 0.0f;
    if (have > 0)
        for (int64_t r = p * chunk + w; r < end; r += 4) {
            const Vec<T, E> vd = load_upto<T, E>(static_cast<const T *>(a.dy) + r * a.dyrs + c, have);
            const Vec<T, E> vx = load_upto<T, E>(static_cast<const T *>(a.x) + r * a.xrs + c, have);
            const float m = a.mean[r], rs = a.rstd[r];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float dy = to_f<T>(vd.v[e]);
                s[e] += dy * ((to_f<T>(vx.v[e]) - m) * rs);
                b[e] += dy;
            }
        }
#pragma unroll
    for (int e = 0; e < E; ++e) sh[0][w][l * E + e] = s[e], sh[1][w][l * E + e] = b[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * 64 * E; i += 256) {
        const int which = i / (64 * E), k = i % (64 * E);
        const int64_t col = (int64_t)blockIdx.x * 64 * E + k;
        if (col < a.cols)
            a.part[(p * 2 + which) * a.cols + col] =
                (sh[which][0][k] + sh[which][1][k]) + (sh[which][2][k] + sh[which][3][k]);
    }
}
template <typename T>
__device__ __forceinline__ void ln_param_planar(const OpsLnBwdArgs &a) {
    __shared__ float sh[8];
    const int64_t c = blockIdx.x, p = blockIdx.y;
    const int64_t chunk = (a.rows + a.nparts - 1) / a.nparts, end = min(a.rows, (p + 1) * chunk);
    float s = 0.0f, b = 0.0f;
    for (int64_t r = p * chunk + threadIdx.x; r < end; r += 256) {
        const float dy = to_f<T>(static_cast<const T *>(a.dy)[c * a.dycs + r]);
        s += dy * ((to_f<T>(static_cast<const T *>(a.x)[c * a.xcs + r]) - a.mean[r]) * a.rstd[r]);
        b += dy;
    }
    s = wave_sum(s);
    b = wave_sum(b);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s, sh[4 + (threadIdx.x >> 6)] = b;
    __syncthreads();
    if (threadIdx.x < 2) {
        const float *v = sh + threadIdx.x * 4;
        a.part[(p * 2 + threadIdx.x) * a.cols + c] = (v[0] + v[1]) + (v[2] + v[3]);
    }
}

// dz = dy act'(z) and the bias's partial sums. Rows with contiguous columns:
// 64 x E columns by a run of rows a block, a wave a row at a time.
template <typename T>
__device__ __forceinline__ void dz_rows(const OpsDzArgs &a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float sh[4][64 * E];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + l) * E, p = blockIdx.y, have = a.cols - c;
    const int64_t chunk = (a.rows + a.nparts - 1) / a.nparts, end = min(a.rows, (p + 1) * chunk);
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
    if (have > 0)
        for (int64_t r = p * chunk + w; r < end; r += 4) {
            Vec<T, E> vd = load_upto<T, E>(static_cast<const T *>(a.dy) + r * a.dyrs + c, have);
            Vec<T, E> vz;
            if (a.z) vz = load_upto<T, E>(static_cast<const T *>(a.z) + r * a.zrs + c, have);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float v = to_f<T>(vd.v[e]);
                if (a.z) v *= act_bwd(a.act, a.slope, to_f<T>(vz.v[e]));
                s[e] += v;
                vd.v[e] = from_f<T>(v);
            }
            if (a.dz) store_upto<T, E>(static_cast<T *>(a.dz) + r * a.drs + c, vd, have);
        }
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < E; ++e) sh[w][l * E + e] = s[e];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * E; k += 256) {
        const int64_t col = (int64_t)blockIdx.x * 64 * E + k;
        if (col < a.cols) a.part[p * a.cols + col] = (sh[0][k] + sh[1][k]) + (sh[2][k] + sh[3][k]);
    }
}
// Planar order: one feature by a run of positions a block.
template <typename T>
__device__ __forceinline__ void dz_planar(const OpsDzArgs &a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float sh[4];
    const int64_t c = blockIdx.x, p = blockIdx.y;
    const int64_t chunk = ((a.rows + a.nparts - 1) / a.nparts + E - 1) / E * E, end = min(a.rows, (p + 1) * chunk);
    float s = 0.0f;
    for (int64_t r = p * chunk + threadIdx.x * E; r < end; r += 256 * E) {
        Vec<T, E> vd = load_upto<T, E>(static_cast<const T *>(a.dy) + c * a.dycs + r, end - r);
        Vec<T, E> vz;
        if (a.z) vz = load_upto<T, E>(static_cast<const T *>(a.z) + c * a.zcs + r, end - r);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float v = to_f<T>(vd.v[e]);
            if (a.z) v *= act_bwd(a.act, a.slope, to_f<T>(vz.v[e]));
            if (r + e < end) s += v;
            vd.v[e] = from_f<T>(v);
        }
        if (a.dz) store_upto<T, E>(static_cast<T *>(a.dz) + c * a.dcs + r, vd, end - r);
    }
    if (!a.part) return;
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[p * a.cols + c] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
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

#define OPS_LN_ROWS(name, T, LPR, NV, BT)                                                                       \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_rows_##name##_##LPR##x##NV(OpsLnArgs a) {            \
        ln_rows<T, LPR, NV, BT>(a);                                                                              \
    }
#define OPS_LN_BWD_ROWS(name, T, LPR, NV, BT)                                                                   \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_bwd_rows_##name##_##LPR##x##NV(OpsLnBwdArgs a) {     \
        ln_bwd_rows<T, LPR, NV, BT>(a);                                                                          \
    }
#define OPS_LN_PLANAR(name, T, BT, CH)                                                                          \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_planar_##name##_##BT##x##CH(OpsLnArgs a) {           \
        ln_planar<T, BT, CH, false>(a);                                                                          \
    }                                                                                                            \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_bwd_planar_##name##_##BT##x##CH(OpsLnBwdArgs a) {    \
        ln_bwd_planar<T, BT, CH, false>(a);                                                                      \
    }
#define OPS_ROWS_TYPE(name, T)                                                                                        \
    OPS_LN_ROWS(name, T, 8, 1, 256)                                                                                   \
    OPS_LN_ROWS(name, T, 16, 1, 256)                                                                                  \
    OPS_LN_ROWS(name, T, 32, 1, 256)                                                                                  \
    OPS_LN_ROWS(name, T, 64, 1, 256)                                                                                  \
    OPS_LN_ROWS(name, T, 64, 2, 256)                                                                                  \
    OPS_LN_ROWS(name, T, 256, 1, 256)                                                                                 \
    OPS_LN_ROWS(name, T, 256, 2, 256)                                                                                 \
    OPS_LN_ROWS(name, T, 1024, 1, 1024)                                                                               \
    OPS_LN_ROWS(name, T, 1024, 2, 1024)                                                                               \
    OPS_LN_BWD_ROWS(name, T, 8, 1, 256)                                                                               \
    OPS_LN_BWD_ROWS(name, T, 16, 1, 256)                                                                              \
    OPS_LN_BWD_ROWS(name, T, 32, 1, 256)                                                                              \
    OPS_LN_BWD_ROWS(name, T, 64, 1, 256)                                                                              \
    OPS_LN_BWD_ROWS(name, T, 64, 2, 256)                                                                              \
    OPS_LN_BWD_ROWS(name, T, 256, 1, 1024)                                                                            \
    OPS_LN_BWD_ROWS(name, T, 256, 2, 1024)                                                                            \
    OPS_LN_BWD_ROWS(name, T, 1024, 1, 1024)                                                                           \
    OPS_LN_BWD_ROWS(name, T, 1024, 2, 1024)                                                                           \
    OPS_LN_PLANAR(name, T, 256, 1)                                                                                    \
    OPS_LN_PLANAR(name, T, 256, 2)                                                                                    \
    OPS_LN_PLANAR(name, T, 256, 4)                                                                                    \
    OPS_LN_PLANAR(name, T, 256, 8)                                                                                    \
    OPS_LN_PLANAR(name, T, 1024, 4)                                                                                   \
    OPS_LN_PLANAR(name, T, 1024, 8)                                                                                   \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_planar_##name##_loop(OpsLnArgs a) {                     \
        ln_planar<T, 1024, 4, true>(a);                                                                               \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_bwd_planar_##name##_loop(OpsLnBwdArgs a) {              \
        ln_bwd_planar<T, 1024, 4, true>(a);                                                                           \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_rows_##name##_long(OpsLnArgs a) { ln_long<T>(a); }      \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_bwd_rows_##name##_long(OpsLnBwdArgs a) {                \
        ln_bwd_long<T>(a);                                                                                            \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void mxo_ln_param_rows_##name(OpsLnBwdArgs a) { ln_param_rows<T>(a); } \
    extern "C" __global__ __launch_bounds__(256) void mxo_ln_param_planar_##name(OpsLnBwdArgs a) {                    \
        ln_param_planar<T>(a);                                                                                        \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void mxo_dz_rows_##name(OpsDzArgs a) { dz_rows<T>(a); }              \
    extern "C" __global__ __launch_bounds__(256) void mxo_dz_planar_##name(OpsDzArgs a) { dz_planar<T>(a); }

OPS_ROWS_TYPE(bf16, bf16)
OPS_ROWS_TYPE(f16, f16)
OPS_ROWS_TYPE(f32, float)
