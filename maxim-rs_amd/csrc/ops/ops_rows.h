// LayerNorm, its backward pass and the activation's derivative with the
// bias's gradient: passes over [rows][cols] activations of either order.
//
// All of them are bound by memory: a row (or, in planar order, a column of 64
// positions) is read once into registers, reduced there, and written from
// there. The gradients of the parameters are sums over all rows: each block
// keeps its own in registers over the rows it walks and writes one partial
// sum, and mxo_join_parts adds those in their order, so the bits do not depend
// on which block ran first.
//
// Against 4.9 TB/s for a large copy: rows of 32 to 16384 16-bit elements go at
// 3.6-5.1 TB/s, of 32 to 8192 floats at 5.2-5.9 (67 MB each way, partly still
// in the 256 MB cache), the backward pass up to 4.9. Planar floats 4.6-6.0,
// backward 3.5-4.6; planar 16-bit channels 3.0-3.8, backward 2.5-3.4: eight
// elements a vector mean as many sums across threads as vectors a lane holds,
// and the registers for them leave fewer loads in flight. Rows and columns
// that registers do not hold are read three times: 1.0-2.9.
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
// parameters are read once a block, which walks over rows with the next one on
// its way: 8192 rows of 4096 bf16, 134 MB, take 32 us (44 with one row at a
// time). WHOLE: rows are whole vectors.
template <typename T, int LPR, int NV, int BT, bool WHOLE>
__device__ __forceinline__ void ln_rows(const OpsLnArgs &a, float *at) {
    constexpr int E = 16 / sizeof(T), RPB = BT / LPR;
    const int li = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const int cols = (int)a.cols;
    const float n = (float)a.cols;
    float sc[NV][E], bi[NV][E];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + li) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sc[j][e] = c + e < cols ? param<T>(a.scale, c + e, a.param_f32) : 0.0f;
            bi[j][e] = a.bias && c + e < cols ? param<T>(a.bias, c + e, a.param_f32) : 0.0f;
        }
    }
    int turn = 0;
    u32x4 ahead[NV];
    auto fetch = [&](int64_t r0) {
        // past the end: the last row again, not stored
        const T *x0 = static_cast<const T *>(a.x), *x = x0 + min(r0 + grp, a.rows - 1) * a.xrs;
        const T *last = x0 + (a.rows - 1) * a.xrs + cols - E;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + li) * E;
            ahead[j] = load_raw<T, E, WHOLE>(x + c, x, last, cols - c);
        }
    };
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    if (r0 < a.rows) fetch(r0);
    for (; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + grp;
        u32x4 v[NV];
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = ahead[j];
        if (r0 + step < a.rows) fetch(r0 + step);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) s += (j * LPR + li) * E + e < cols ? elem<T>(v[j], e) : 0.0f;
        float zero = 0.0f;
        row_sum2<LPR, BT>(s, zero, at, turn++);
        const float mean = s / n;  // a division: the mean of equal values is that value
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = elem<T>(v[j], e) - mean;
                q += (j * LPR + li) * E + e < cols ? d * d : 0.0f;
            }
        zero = 0.0f;
        row_sum2<LPR, BT>(q, zero, at, turn++);
        const float rstd = 1.0f / sqrtf(q / n + a.eps);
        if (r >= a.rows) continue;  // behind the round's last barrier
        T *y = static_cast<T *>(a.y) + r * a.yrs;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + li) * E;
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.v[e] = from_f<T>((elem<T>(v[j], e) - mean) * rstd * sc[j][e] + bi[j][e]);
            store_in<T, E, WHOLE>(y + c, o, cols - c);
        }
        if (li == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// The backward pass in the same arrangement: dx from registers, the
// parameters' gradients summed in registers over the block's rows, then over
// its row groups in LDS. With one vector a thread the next row's are loaded
// before the present row's sums, whose barrier a large block's waves share;
// two vectors leave no registers for that, nor, of 16-bit elements, for the
// parameters' sums (PARAMS off: those are another launch's; with them 4096 rows
// of 16384 bf16 spilled and took 422 us). 8192 rows of 4096 bf16, 268 MB: 51 us
// and 5 for joining the blocks' sums.
template <typename T, int LPR, int NV, int BT, bool PARAMS, bool WHOLE>
__device__ __forceinline__ void ln_bwd_rows(const OpsLnBwdArgs &a, float *at, float *sums) {
    constexpr int E = 16 / sizeof(T), RPB = BT / LPR;
    constexpr bool KEEP = NV == 1;  // the scale in registers; two vectors' would not leave room
    const int li = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const int cols = (int)a.cols;
    const float n = (float)a.cols;
    float sc[KEEP ? E : 1], ds[NV][E], db[NV][E];
    if constexpr (KEEP)
#pragma unroll
        for (int e = 0; e < E; ++e) sc[e] = li * E + e < cols ? param<T>(a.scale, li * E + e, a.param_f32) : 0.0f;
    auto scale = [&](int j, int e) {
        if constexpr (KEEP) return sc[e];
        const int c = (j * LPR + li) * E + e;
        return c < cols ? param<T>(a.scale, c, a.param_f32) : 0.0f;
    };
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) ds[j][e] = db[j][e] = 0.0f;
    u32x4 vx[NV], vd[NV], va[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](int64_t r0) {
        const int64_t r = min(r0 + grp, a.rows - 1);  // past the end: the last row again, not stored
        const T *x = static_cast<const T *>(a.x) + r * a.xrs, *dy = static_cast<const T *>(a.dy) + r * a.dyrs;
        const T *add = static_cast<const T *>(a.add) + r * a.ars;
        const int64_t on = a.rows - 1 - r, end = cols - E;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + li) * E;
            vx[j] = load_raw<T, E, WHOLE>(x + c, x, x + on * a.xrs + end, cols - c);
            vd[j] = load_raw<T, E, WHOLE>(dy + c, dy, dy + on * a.dyrs + end, cols - c);
            if (a.add) va[j] = load_raw<T, E, WHOLE>(add + c, add, add + on * a.ars + end, cols - c);
        }
        mean = a.mean[r];
        rstd = a.rstd[r];
    };
    const int64_t step = (int64_t)gridDim.x * RPB;
    int turn = 0;
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    if (KEEP && r0 < a.rows) fetch(r0);
    for (; r0 < a.rows; r0 += step) {
        const bool on = r0 + grp < a.rows;
        if (!KEEP) fetch(r0);
        u32x4 cx[NV], cd[NV], ca[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) cx[j] = vx[j], cd[j] = vd[j], ca[j] = va[j];
        const float m = mean, rs = rstd;
        if (KEEP && r0 + step < a.rows) fetch(r0 + step);
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool in = on && (j * LPR + li) * E + e < cols;
                const float dy = in ? elem<T>(cd[j], e) : 0.0f;
                const float xh = in ? (elem<T>(cx[j], e) - m) * rs : 0.0f;
                const float g = dy * scale(j, e);
                s += g;
                q += g * xh;
                if (PARAMS) ds[j][e] += dy * xh, db[j][e] += dy;
            }
        if (!a.dx) continue;
        row_sum2<LPR, BT>(s, q, at, turn++);
        s /= n;
        q /= n;
        if (!on) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (NV > 1) reread(cx[j]), reread(cd[j]);
        T *dx = static_cast<T *>(a.dx) + (r0 + grp) * a.dxrs;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + li) * E;
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xh = (elem<T>(cx[j], e) - m) * rs;
                float v = rs * (elem<T>(cd[j], e) * scale(j, e) - s - xh * q);
                if (a.add) v += elem<T>(ca[j], e);
                o.v[e] = from_f<T>(v);
            }
            store_in<T, E, WHOLE>(dx + c, o, cols - c);
        }
    }
    if (!PARAMS || !a.part) return;
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
            for (int i = threadIdx.x; i < LPR * NV * E && i < cols; i += BT) {
                float s = 0.0f;
#pragma unroll 4
                for (int g = 0; g < RPB; ++g) s += sums[g * (LPR * NV * E) + i];
                part[which * a.cols + i] = s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * LPR + li) * E;
                Vec<float, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = which ? db[j][e] : ds[j][e];
                store_upto<float, E>(part + which * a.cols + c, o, cols - c);
            }
        }
    }
}

// Planar order: LP lanes of 16 bytes along the positions, S = BT / LP threads
// down the channels, CH channels a thread, all in registers. Sums over channels
// run over a thread's own, the wave's lanes and, through LDS, the block's
// waves. Many lanes along the positions leave little to add across threads:
// 32 bf16 channels of 2^21 pixels took 151 us with 8 lanes, 78 with 64. 64 fp32
// channels of 448 x 640, 147 MB, take 31 us; backward 32, 110 MB, 24 us.
template <typename T, int BT, int LP>
struct PlanarTile {
    static constexpr int E = 16 / sizeof(T), S = BT / LP, W = BT / 64, POS = LP * E;
    // N sums for each of a thread's E positions, over the block's channels;
    // `at` holds N * W * POS floats
    template <int N>
    static __device__ __forceinline__ void sum(float (&v)[N][E], float *at) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int o = LP; o < 64; o <<= 1) v[n][e] += __shfl_xor(v[n][e], o);
        __syncthreads();
        if (lane < LP)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<f32x4 *>(at + (n * W + w) * POS + lane * E + e) =
                        f32x4{v[n][e], v[n][e + 1], v[n][e + 2], v[n][e + 3]};
        __syncthreads();
        const int p = (lane % LP) * E;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
                for (int i = 0; i < W; ++i) s += *reinterpret_cast<const f32x4 *>(at + (n * W + i) * POS + p + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[n][e + k] = s[k];
            }
    }
};

// (Addresses are the lane's own part plus the channel's, worked out in the
// scalar unit for each tile, which here() sees to: kept over the tiles they
// would take more registers than the data.)
// LOOP: any number of channels, read again for each of the three passes.
// WHOLE: the positions are whole vectors.
template <typename T, int BT, int LP, int CH, bool LOOP, bool WHOLE>
__device__ __forceinline__ void ln_planar(const OpsLnArgs &a, float *at) {
    typedef PlanarTile<T, BT, LP> P;
    constexpr int E = P::E, S = P::S;
    const int pl = threadIdx.x % LP, sl = threadIdx.x / LP;
    const float n = (float)a.cols;
    const int rounds = LOOP ? (int)((a.cols + S * CH - 1) / (S * CH)) : 1;
    const T *x = static_cast<const T *>(a.x), *xl = x + (a.cols - 1) * a.xcs + a.rows - E;
    for (int64_t p0 = (int64_t)blockIdx.x * P::POS; p0 < a.rows; p0 += (int64_t)gridDim.x * P::POS) {
        const int64_t sx = here(S * a.xcs), sy = here(S * a.ycs);
        const int64_t p = p0 + pl * E, have = a.rows - p;
        u32x4 v[CH];
        auto fetch = [&](int round) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                v[j] = load_in<T, E, WHOLE>(x + (sl * a.xcs + p) + (round * CH + j) * sx, x, xl, c < a.cols ? have : 0);
            }
        };
        float s[1][E], q[1][E];
#pragma unroll
        for (int e = 0; e < E; ++e) s[0][e] = q[0][e] = 0.0f;
        for (int round = 0; round < rounds; ++round) {
            fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) s[0][e] += elem<T>(v[j], e);
        }
        P::sum(s, at);
#pragma unroll
        for (int e = 0; e < E; ++e) s[0][e] /= n;
        for (int round = 0; round < rounds; ++round) {
            if (LOOP) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                reread(v[j]);
                const bool in = ((int64_t)round * CH + j) * S + sl < a.cols;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = elem<T>(v[j], e) - s[0][e];
                    q[0][e] += in ? d * d : 0.0f;
                }
            }
        }
        P::sum(q, at);
#pragma unroll
        for (int e = 0; e < E; ++e) q[0][e] = 1.0f / sqrtf(q[0][e] / n + a.eps);
        for (int round = 0; round < rounds; ++round) {
            if (LOOP) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                reread(v[j]);
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                if (c >= a.cols) continue;
                const float sc = param<T>(a.scale, c, a.param_f32), bi = a.bias ? param<T>(a.bias, c, a.param_f32) : 0.0f;
                Vec<T, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = from_f<T>((elem<T>(v[j], e) - s[0][e]) * q[0][e] * sc + bi);
                store_in<T, E, WHOLE>(static_cast<T *>(a.y) + (sl * a.ycs + p) + (round * CH + j) * sy, o, have);
            }
        }
        if (sl == 0) {
            Vec<float, E> m, r;
#pragma unroll
            for (int e = 0; e < E; ++e) m.v[e] = s[0][e], r.v[e] = q[0][e];
            if (a.mean) store_upto<float, E>(a.mean + p, m, have);
            if (a.rstd) store_upto<float, E>(a.rstd + p, r, have);
        }
    }
}

template <typename T, int BT, int LP, int CH, bool LOOP, bool WHOLE>
__device__ __forceinline__ void ln_bwd_planar(const OpsLnBwdArgs &a, float *at) {
    typedef PlanarTile<T, BT, LP> P;
    constexpr int E = P::E, S = P::S;
    const int pl = threadIdx.x % LP, sl = threadIdx.x / LP;
    const float n = (float)a.cols;
    const int rounds = LOOP ? (int)((a.cols + S * CH - 1) / (S * CH)) : 1;
    const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy), *add = static_cast<const T *>(a.add);
    const T *xl = x + (a.cols - 1) * a.xcs + a.rows - E, *dyl = dy + (a.cols - 1) * a.dycs + a.rows - E;
    const T *addl = add + (a.cols - 1) * a.acs + a.rows - E;
    float ds[CH], db[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) ds[j] = db[j] = 0.0f;
    for (int64_t p0 = (int64_t)blockIdx.x * P::POS; p0 < a.rows; p0 += (int64_t)gridDim.x * P::POS) {
        const int64_t sx = here(S * a.xcs), sdy = here(S * a.dycs), sa = here(S * a.acs), sdx = here(S * a.dxcs);
        const int64_t p = p0 + pl * E, have = a.rows - p;
        u32x4 vx[CH], vd[CH];
        auto fetch = [&](int round) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl, left = c < a.cols ? have : 0;
                vx[j] = load_in<T, E, WHOLE>(x + (sl * a.xcs + p) + (round * CH + j) * sx, x, xl, left);
                vd[j] = load_in<T, E, WHOLE>(dy + (sl * a.dycs + p) + (round * CH + j) * sdy, dy, dyl, left);
            }
        };
        fetch(0);
        // past the last position rstd is 0, so what lies there adds nothing
        const Vec<float, E> m = load_upto<float, E>(a.mean + p, have), r = load_upto<float, E>(a.rstd + p, have);
        float sum[2][E];  // of g and of g xh
#pragma unroll
        for (int e = 0; e < E; ++e) sum[0][e] = sum[1][e] = 0.0f;
        for (int round = 0; round < rounds; ++round) {
            if (round) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                const bool in = c < a.cols;
                const float sc = in ? param<T>(a.scale, c, a.param_f32) : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = elem<T>(vd[j], e);
                    const float xh = in ? (elem<T>(vx[j], e) - m.v[e]) * r.v[e] : 0.0f;
                    sum[0][e] += d * sc;
                    sum[1][e] += d * sc * xh;
                    if (!LOOP) ds[j] += d * xh, db[j] += d;
                }
                // one channel's elements as fp32 at a time
                if (CH >= 8) __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!a.dx) continue;
        P::sum(sum, at);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[0][e] /= n, sum[1][e] /= n;
#pragma unroll
        for (int j = 0; j < CH; ++j) reread(vx[j]), reread(vd[j]);
        for (int round = 0; round < rounds; ++round) {
            if (LOOP) fetch(round);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int64_t c = ((int64_t)round * CH + j) * S + sl;
                if (c >= a.cols) continue;
                const float sc = param<T>(a.scale, c, a.param_f32);
                Vec<T, E> o;
                u32x4 va;
                if (a.add) va = load_in<T, E, WHOLE>(add + (sl * a.acs + p) + (round * CH + j) * sa, add, addl, have);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float xh = (elem<T>(vx[j], e) - m.v[e]) * r.v[e];
                    float v = r.v[e] * (elem<T>(vd[j], e) * sc - sum[0][e] - xh * sum[1][e]);
                    if (a.add) v += elem<T>(va, e);
                    o.v[e] = from_f<T>(v);
                }
                store_in<T, E, WHOLE>(static_cast<T *>(a.dx) + (sl * a.dxcs + p) + (round * CH + j) * sdx, o, have);
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
    constexpr int E = 16 / sizeof(T);
    __shared__ float at[16];
    const float n = (float)a.cols;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.xrs;
        const T *xl = x + (a.rows - 1 - r) * a.xrs + a.cols - E;
        T *y = static_cast<T *>(a.y) + r * a.yrs;
        float s = 0.0f;
        for (int64_t c = threadIdx.x * E; c < a.cols; c += 1024 * E) {
            const u32x4 v = load_in<T, E, false>(x + c, x, xl, a.cols - c);
#pragma unroll
            for (int e = 0; e < E; ++e) s += elem<T>(v, e);
        }
        const float mean = block_sum(s, at) / n;
        s = 0.0f;
        for (int64_t c = threadIdx.x * E; c < a.cols; c += 1024 * E) {
            const u32x4 v = load_in<T, E, false>(x + c, x, xl, a.cols - c);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = elem<T>(v, e) - mean;
                s += c + e < a.cols ? d * d : 0.0f;
            }
        }
        const float rstd = 1.0f / sqrtf(block_sum(s, at) / n + a.eps);
        for (int64_t c = threadIdx.x * E; c < a.cols; c += 1024 * E) {
            const u32x4 v = load_in<T, E, false>(x + c, x, xl, a.cols - c);
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (c + e >= a.cols) continue;
                const float b = a.bias ? param<T>(a.bias, c + e, a.param_f32) : 0.0f;
                o.v[e] = from_f<T>((elem<T>(v, e) - mean) * rstd * param<T>(a.scale, c + e, a.param_f32) + b);
            }
            store_upto<T, E>(y + c, o, a.cols - c);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__device__ __forceinline__ void ln_bwd_long(const OpsLnBwdArgs &a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float at[16];
    const float n = (float)a.cols;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.xrs;
        const T *dy = static_cast<const T *>(a.dy) + r * a.dyrs;
        const T *add = a.add ? static_cast<const T *>(a.add) + r * a.ars : nullptr;
        T *dx = static_cast<T *>(a.dx) + r * a.dxrs;
        const int64_t rest = a.rows - 1 - r, end = a.cols - E;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s = 0.0f, q = 0.0f;
        for (int64_t c = threadIdx.x * E; c < a.cols; c += 1024 * E) {
            const u32x4 vx = load_in<T, E, false>(x + c, x, x + rest * a.xrs + end, a.cols - c);
            const u32x4 vd = load_in<T, E, false>(dy + c, dy, dy + rest * a.dyrs + end, a.cols - c);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (c + e >= a.cols) continue;
                const float gr = elem<T>(vd, e) * param<T>(a.scale, c + e, a.param_f32);
                s += gr;
                q += gr * ((elem<T>(vx, e) - mean) * rstd);
            }
        }
        s = block_sum(s, at) / n;
        q = block_sum(q, at) / n;
        for (int64_t c = threadIdx.x * E; c < a.cols; c += 1024 * E) {
            const u32x4 vx = load_in<T, E, false>(x + c, x, x + rest * a.xrs + end, a.cols - c);
            const u32x4 vd = load_in<T, E, false>(dy + c, dy, dy + rest * a.dyrs + end, a.cols - c);
            u32x4 va;
            Vec<T, E> o;
            if (add) va = load_in<T, E, false>(add + c, add, add + rest * a.ars + end, a.cols - c);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (c + e >= a.cols) continue;
                const float gr = elem<T>(vd, e) * param<T>(a.scale, c + e, a.param_f32);
                float v = rstd * (gr - s - (elem<T>(vx, e) - mean) * rstd * q);
                if (add) v += elem<T>(va, e);
                o.v[e] = from_f<T>(v);
            }
            store_upto<T, E>(dx + c, o, a.cols - c);
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
            const T *dy = static_cast<const T *>(a.dy) + r * a.dyrs + c, *x = static_cast<const T *>(a.x) + r * a.xrs + c;
            const int64_t rest = a.rows - 1 - r, end = a.cols - E - c;
            const u32x4 vd = load_in<T, E, false>(dy, dy, dy + rest * a.dyrs + end, have);
            const u32x4 vx = load_in<T, E, false>(x, x, x + rest * a.xrs + end, have);
            const float m = a.mean[r], rs = a.rstd[r];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = elem<T>(vd, e);
                s[e] += e < have ? d * ((elem<T>(vx, e) - m) * rs) : 0.0f;
                b[e] += d;
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
// 64 x E columns by a run of rows a block, a wave a row at a time: 4096 x 4096
// bf16, 101 MB, 22 us. (A pass of its own because both products read dz, each
// tile of it many times: formed inside them it would be formed again each time.)
// It is stored rounded to the operands' type, as the matrix cores take it: two
// parts of 16 bits each would double both products. That half step a term shows
// in dx and dw (4096 x 1024 to 4096 bf16: relative errors 2.3e-3 against 64 bits,
// 1.7e-3 with dz in fp32); the bias's sums take dz before the rounding.
template <typename T, bool WHOLE>
__device__ __forceinline__ void dz_rows(const OpsDzArgs &a, float (*sh)[64 * 16 / sizeof(T)]) {
    constexpr int E = 16 / sizeof(T);
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + l) * E, p = blockIdx.y, have = a.cols - c;
    const int64_t chunk = (a.rows + a.nparts - 1) / a.nparts, end = min(a.rows, (p + 1) * chunk);
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.0f;
    if (have > 0)
        for (int64_t r = p * chunk + w; r < end; r += 4) {
            const T *dy = static_cast<const T *>(a.dy) + r * a.dyrs + c, *z = static_cast<const T *>(a.z) + r * a.zrs + c;
            // a lane without columns has left already
            const int64_t rest = a.rows - 1 - r, end = a.cols - E - c;
            const u32x4 vd = load_in<T, E, WHOLE>(dy, dy, dy + rest * a.dyrs + end, have);
            u32x4 vz;
            if (a.z) vz = load_in<T, E, WHOLE>(z, z, z + rest * a.zrs + end, have);
            float v[E];
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = elem<T>(vd, e);
            if (a.z) act_bwd_n<E>(a.act, a.slope, v, [&](int e) { return elem<T>(vz, e); });
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s[e] += v[e];
                o.v[e] = from_f<T>(v[e]);
            }
            // lines of dz are whole vectors, their ends zeros
            if (a.dz) store_n<T, E>(static_cast<T *>(a.dz) + r * a.drs + c, o);
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
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = to_f<T>(vd.v[e]);
        if (a.z) act_bwd_n<E>(a.act, a.slope, v, [&](int e) { return to_f<T>(vz.v[e]); });
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (r + e < end) s += v[e];
            vd.v[e] = from_f<T>(v[e]);
        }
        // lines of dz are whole vectors, their ends zeros (a run is whole vectors)
        if (a.dz) store_n<T, E>(static_cast<T *>(a.dz) + c * a.dcs + r, vd);
    }
    if (!a.part) return;
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.part[p * a.cols + c] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__device__ __forceinline__ void join_store(void *out, int dtype, int64_t i, float v) {
    if (dtype == MXO_F32) static_cast<float *>(out)[i] = v;
    else if (dtype == MXO_F16) static_cast<f16 *>(out)[i] = from_f<f16>(v);
    else static_cast<bf16 *>(out)[i] = from_f<bf16>(v);
}
// Partial sums added in a fixed order: 16 columns a block, 64 threads down
// the parts, eight loads in flight each, then a tree over the 64 in LDS. (64
// columns a block walked 1024 parts of 32 columns in 17 us, this in 4.)
extern "C" __global__ __launch_bounds__(1024) void mxo_join_parts(OpsJoinArgs a) {
    __shared__ float sh[64][17];
    const int l = threadIdx.x & 15, w = threadIdx.x >> 4, which = blockIdx.y;
    const int64_t c = (int64_t)blockIdx.x * 16 + l;
    float s = 0.0f;
    if (c < a.n) {
        const float *p = a.part + which * a.n + c;
        const int64_t step = (int64_t)a.nout * a.n;
#pragma unroll 8
        for (int i = w; i < a.nparts; i += 64) s += p[i * step];
    }
    sh[w][l] = s;
#pragma unroll
    for (int half = 32; half >= 1; half >>= 1) {
        __syncthreads();
        if (w < half) sh[w][l] += sh[w + half][l];
    }
    if (w == 0 && c < a.n) join_store(which ? a.out1 : a.out0, a.dtype, c, sh[0][l]);
}

// Each kernel has both forms, of whole vectors and of any number of elements.
#define OPS_BOTH(extent, E, call_whole, call_any) \
    if ((extent) % (E) == 0) call_whole;          \
    else call_any;

#define OPS_LN_ROWS(name, T, LPR, NV, BT)                                                                             \
    extern "C" __global__ __launch_bounds__(BT, NV == 1 ? 8 : 4) void mxo_ln_rows_##name##_##LPR##x##NV(OpsLnArgs a) { \
        __shared__ float at[4 * (BT / 64)];                                                                           \
        OPS_BOTH(a.cols, 16 / sizeof(T), (ln_rows<T, LPR, NV, BT, true>(a, at)), (ln_rows<T, LPR, NV, BT, false>(a, at))) \
    }
#define OPS_LN_BWD_ROWS(name, T, LPR, NV, BT)                                                                         \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_bwd_rows_##name##_##LPR##x##NV(OpsLnBwdArgs a) {          \
        __shared__ float at[4 * (BT / 64)];                                                                           \
        __shared__ float sums[BT > LPR ? BT * NV * 16 / sizeof(T) : 1];                                               \
        constexpr bool P = NV == 1 || sizeof(T) == 4;                                                                 \
        OPS_BOTH(a.cols, 16 / sizeof(T), (ln_bwd_rows<T, LPR, NV, BT, P, true>(a, at, sums)),                         \
                 (ln_bwd_rows<T, LPR, NV, BT, P, false>(a, at, sums)))                                                \
    }
#define OPS_LN_FWD_PLANAR1(name, T, tag, BT, LP, CH, LOOP)                                                            \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_planar_##name##_##tag(OpsLnArgs a) {                      \
        __shared__ __align__(16) float at[BT / 64 * LP * 16 / sizeof(T)];                                             \
        OPS_BOTH(a.rows, 16 / sizeof(T), (ln_planar<T, BT, LP, CH, LOOP, true>(a, at)),                               \
                 (ln_planar<T, BT, LP, CH, LOOP, false>(a, at)))                                                      \
    }
#define OPS_LN_BWD_PLANAR1(name, T, tag, BT, LP, CH, LOOP)                                                            \
    extern "C" __global__ __launch_bounds__(BT) void mxo_ln_bwd_planar_##name##_##tag(OpsLnBwdArgs a) {               \
        __shared__ __align__(16) float at[2 * BT / 64 * LP * 16 / sizeof(T)];                                         \
        OPS_BOTH(a.rows, 16 / sizeof(T), (ln_bwd_planar<T, BT, LP, CH, LOOP, true>(a, at)),                           \
                 (ln_bwd_planar<T, BT, LP, CH, LOOP, false>(a, at)))                                                  \
    }
#define OPS_LN_FWD_PLANAR(name, T, BT, LP, CH) OPS_LN_FWD_PLANAR1(name, T, BT##x##LP##x##CH, BT, LP, CH, false)
#define OPS_LN_BWD_PLANAR(name, T, BT, LP, CH) OPS_LN_BWD_PLANAR1(name, T, BT##x##LP##x##CH, BT, LP, CH, false)
#define OPS_LN_BOTH(name, T, LPR, NV, BT) \
    OPS_LN_ROWS(name, T, LPR, NV, BT)     \
    OPS_LN_BWD_ROWS(name, T, LPR, NV, BT)
#define OPS_ROWS_TYPE(name, T)                                                                                        \
    OPS_LN_BOTH(name, T, 8, 1, 256)                                                                                   \
    OPS_LN_BOTH(name, T, 16, 1, 256)                                                                                  \
    OPS_LN_BOTH(name, T, 32, 1, 256)                                                                                  \
    OPS_LN_BOTH(name, T, 64, 1, 256)                                                                                  \
    OPS_LN_ROWS(name, T, 128, 1, 256)                                                                                 \
    OPS_LN_ROWS(name, T, 256, 1, 256)                                                                                 \
    OPS_LN_ROWS(name, T, 512, 1, 512)                                                                                 \
    OPS_LN_BWD_ROWS(name, T, 128, 1, 1024)                                                                            \
    OPS_LN_BWD_ROWS(name, T, 256, 1, 1024)                                                                            \
    OPS_LN_BWD_ROWS(name, T, 512, 1, 1024)                                                                            \
    OPS_LN_BOTH(name, T, 1024, 1, 1024)                                                                               \
    OPS_LN_BOTH(name, T, 1024, 2, 1024)                                                                               \
    OPS_LN_FWD_PLANAR(name, T, 256, 64, 4)                                                                            \
    OPS_LN_FWD_PLANAR(name, T, 256, 64, 8)                                                                            \
    OPS_LN_FWD_PLANAR(name, T, 512, 32, 16)                                                                           \
    OPS_LN_FWD_PLANAR(name, T, 512, 16, 2)                                                                            \
    OPS_LN_FWD_PLANAR(name, T, 512, 16, 4)                                                                            \
    OPS_LN_FWD_PLANAR(name, T, 512, 16, 8)                                                                            \
    OPS_LN_FWD_PLANAR(name, T, 512, 16, 16)                                                                           \
    OPS_LN_FWD_PLANAR(name, T, 512, 8, 16)                                                                            \
    OPS_LN_BWD_PLANAR(name, T, 256, 64, 4)                                                                            \
    OPS_LN_BWD_PLANAR(name, T, 512, 64, 4)                                                                            \
    OPS_LN_BWD_PLANAR(name, T, 512, 16, 1)                                                                            \
    OPS_LN_BWD_PLANAR(name, T, 512, 16, 2)                                                                            \
    OPS_LN_BWD_PLANAR(name, T, 512, 16, 4)                                                                            \
    OPS_LN_FWD_PLANAR1(name, T, loop, 512, 16, 4, true)                                                               \
    OPS_LN_BWD_PLANAR1(name, T, loop, 512, 16, 4, true)                                                               \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_rows_##name##_long(OpsLnArgs a) { ln_long<T>(a); }      \
    extern "C" __global__ __launch_bounds__(1024) void mxo_ln_bwd_rows_##name##_long(OpsLnBwdArgs a) {                \
        ln_bwd_long<T>(a);                                                                                            \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void mxo_ln_param_rows_##name(OpsLnBwdArgs a) { ln_param_rows<T>(a); } \
    extern "C" __global__ __launch_bounds__(256) void mxo_ln_param_planar_##name(OpsLnBwdArgs a) {                    \
        ln_param_planar<T>(a);                                                                                        \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void mxo_dz_rows_##name(OpsDzArgs a) {                               \
        __shared__ float sh[4][64 * 16 / sizeof(T)];                                                                  \
        OPS_BOTH(a.cols, 16 / sizeof(T), (dz_rows<T, true>(a, sh)), (dz_rows<T, false>(a, sh)))                       \
    }                                                                                                                 \
    extern "C" __global__ __launch_bounds__(256) void mxo_dz_planar_##name(OpsDzArgs a) { dz_planar<T>(a); }

OPS_ROWS_TYPE(bf16, bf16)
OPS_ROWS_TYPE(f16, f16)
OPS_ROWS_TYPE(f32, float)
OPS_LN_FWD_PLANAR(f32, float, 512, 64, 16)
OPS_LN_BWD_PLANAR(f32, float, 512, 64, 8)
OPS_LN_BWD_PLANAR(f32, float, 512, 16, 8)
OPS_LN_BWD_PLANAR(f32, float, 512, 8, 8)
OPS_LN_FWD_PLANAR(bf16, bf16, 256, 64, 16)
OPS_LN_FWD_PLANAR(f16, f16, 256, 64, 16)
OPS_LN_FWD_PLANAR(bf16, bf16, 512, 16, 1)
OPS_LN_FWD_PLANAR(f16, f16, 512, 16, 1)
OPS_LN_BWD_PLANAR(bf16, bf16, 512, 32, 4)
OPS_LN_BWD_PLANAR(f16, f16, 512, 32, 4)
OPS_LN_BWD_PLANAR(bf16, bf16, 512, 8, 4)
OPS_LN_BWD_PLANAR(f16, f16, 512, 8, 4)
