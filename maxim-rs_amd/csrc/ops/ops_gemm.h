// Matrix products of the Dense operators on the matrix cores.
//
// One block computes a BM x BN tile of C over a range of k. Both operands'
// tiles go through LDS, 128 bytes of k at a time (64 16-bit elements or 32
// floats), in two buffers: the next tile's loads are in flight while the
// present one is multiplied. Either operand may be contiguous along k or
// along its other axis, so no product of a forward or backward pass needs a
// transposed copy: a 16-bit operand that is not contiguous along k is
// transposed by ds_read_b64_tr_b16 on its way out of LDS, and an fp32 one is
// read element by element, beside the splitting of what has been read and six
// matrix instructions where 16 bits take one.
//
// The MFMA takes B's rows as its own A operand, so that a lane ends up with
// four consecutive n of one m and C is written four elements at a time.
#pragma once

#include "ops_common.h"

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    typedef bf16x8 Frag;
    static __device__ __forceinline__ f32x4 go(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<f16> {
    typedef f16x8 Frag;
    static __device__ __forceinline__ f32x4 go(Frag a, Frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<float> {
    typedef f32x4 Frag;  // four k's of the lane's group, one MFMA each
    static __device__ __forceinline__ f32x4 go(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = mfma16(a[e], b[e], c);
        return c;
    }
};

typedef __attribute__((address_space(3))) char LdsChar;

// One operand's tile: ROWS of m (or n) by 128 bytes of k, in 16-byte chunks
// at LDS positions p * 16. Contiguous along k: position p holds row p / 8, a
// chunk of its 8 picked by exclusive or with the row, so the 16 rows a
// fragment takes at one k fall into different banks. Contiguous along rows:
// position p holds one k's chunk, 16-element segments exchanged likewise.
template <typename T, bool KMAJ, int ROWS, int NT>
struct Tile {
    static constexpr int E = 16 / sizeof(T);    // elements a chunk
    static constexpr int BK = 128 / sizeof(T);  // k's a tile
    static constexpr int CHUNKS = ROWS * 8;
    static constexpr int PER = CHUNKS / NT;     // chunks a thread brings
    static constexpr int CPR = ROWS / E;        // chunks a k, contiguous along rows
    static constexpr int G = sizeof(T);         // chunks a 16-element segment
    static_assert(CHUNKS % NT == 0, "");
    typedef Vec<T, E> Chunk;

    static __device__ __forceinline__ int kswz(int k) {
        return sizeof(T) == 2 ? (k & 3) | ((k >> 3) & 1) << 2 : (k >> 3) & 3;
    }
    // what position p holds: (row, k) of its chunk's first element
    static __device__ __forceinline__ void where(int p, int &row, int &k) {
        if (KMAJ) {
            row = p >> 3;
            k = ((p & 7) ^ ((row >> 1) & 7)) * E;
        } else {
            k = p / CPR;
            const int c = p % CPR;
            row = ((((c / G) ^ (kswz(k) & (ROWS / 16 - 1))) * G) + c % G) * E;
        }
    }
    // the chunk of position p from global memory: zeros past the operand's
    // `rows` rows and `kn` k's (g points at the tile's first element). INSIDE:
    // the tile's k's and, contiguous along rows, its rows are all there; rows
    // past the last may then be any row's (what they give is not stored).
    template <bool INSIDE>
    static __device__ __forceinline__ Chunk load(const T *g, int64_t ld, int p, int rows, int kn) {
        int row, k;
        where(p, row, k);
        if constexpr (INSIDE) return load_n<T, E>(g + (KMAJ ? min(row, rows - 1) * ld + k : k * ld + row));
        const int have = KMAJ ? (row < rows ? kn - k : 0) : (k < kn ? rows - row : 0);
        return load_upto<T, E>(g + (KMAJ ? row * ld + k : k * ld + row), have);
    }
    static __device__ __forceinline__ bool inside(int rows, int kn) { return kn >= BK && (KMAJ || rows == ROWS); }
    // All of a thread's chunks. (One branch for the tile: with one a chunk each
    // load was waited for before the next.)
    static __device__ __forceinline__ void fetch(Chunk (&c)[PER], const T *g, int64_t ld, int t, int rows, int kn) {
        if (inside(rows, kn)) {
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = load<true>(g, ld, i * NT + t, rows, kn);
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = load<false>(g, ld, i * NT + t, rows, kn);
        }
    }
    // Where lane l's part of a fragment lies, but for the fragment's own
    // constants: rows [base, base + 16), row l % 16 of them; k's 8 (l / 16) +
    // 0..7 of 32, which are half a tile (16-bit) or all of it (fp32). The
    // swizzles are exclusive ors of address bits that nothing else of the
    // lane's part uses, so a fragment is one more.
    static __device__ __forceinline__ int lane_part(int l) {
        const int r = l & 15, g = l >> 4;
        if constexpr (KMAJ) {
            return r * 128 + (((sizeof(T) == 2 ? g : 2 * g) ^ ((r >> 1) & 7)) << 4);
        } else if constexpr (sizeof(T) == 2) {
            // each group of 16 lanes reads a 4 x 16 block of (k, row) and
            // gets it back with lane i holding row i's four k's
            const int k = g * 8 + (r >> 2);
            return k * (ROWS * 2) + ((kswz(k) & (ROWS / 16 - 1)) << 5) + (r & 3) * 8;
        } else {
            return g * 8 * (ROWS * 4) + ((g & (ROWS / 16 - 1)) << 6) + r * 4;
        }
    }
    // kk: which half of a 16-bit tile
    static __device__ __forceinline__ typename Mma<T>::Frag frag(const LdsChar *lds, int base, int kk, int part) {
        static_assert(sizeof(T) == 2, "");
        if constexpr (KMAJ) {
            typedef const __attribute__((address_space(3))) typename Mma<T>::Frag *FP;
            return *(FP)(lds + ((part ^ (kk << 6)) + base * 128));
        } else {
            typedef __attribute__((address_space(3))) i16x4 *LP;
            const int at = (part ^ (base << 1)) + kk * 32 * (ROWS * 2);
            const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(lds + at));
            const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)(lds + (at + 4 * ROWS * 2)));
            const i16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(typename Mma<T>::Frag, v);
        }
    }
    static __device__ __forceinline__ void floats(const LdsChar *lds, int base, int part, float (&v)[8]) {
        static_assert(sizeof(T) == 4, "");
        if constexpr (KMAJ) {
            typedef const __attribute__((address_space(3))) f32x4 *FP;
            const f32x4 lo = *(FP)(lds + (part + base * 128)), hi = *(FP)(lds + ((part ^ 16) + base * 128));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
        } else {
            const int at = part ^ (base << 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = *(const __attribute__((address_space(3))) float *)(lds + (at + e * ROWS * 4));
        }
    }
};

// One tile of fp32 operands: three bf16 parts a float and six products of them
// (common.h has the method, its precision and its range), or, exactly as fp32
// products go, fp32 MFMAs. The six take 96 cycles of a SIMD where the fp32
// ones take 256. The splitting, 4.5 vector operations an element, runs beside
// the products of another wave: 4096^3 takes 722-814 us (169-190 TFLOP/s, the
// library's fp32 product 139-151; with fp32 MFMAs here 970), and putting each row's splitting between the row before's products
// made it 785, shifts and subtractions for the dot products changed nothing.
struct Split {
    u32x4 h, m, l;
};
__device__ __forceinline__ Split split8(const float (&v)[8]) {
    Split s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h, m, l;
        split2(v[2 * i] * kSplitScale, v[2 * i + 1] * kSplitScale, h, m, l);
        s.h[i] = h, s.m[i] = m, s.l[i] = l;
    }
    return s;
}
template <typename TA, typename TB, int FM, int FN>
__device__ __forceinline__ void split_tile(const LdsChar *at, const LdsChar *bt, int wm, int wn, int pa, int pb,
                                           f32x4 (&acc)[FM][FN]) {
    float v[8];
    Split b[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        TB::floats(bt, wn + j * 16, pb, v);
        b[j] = split8(v);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        TA::floats(at, wm + i * 16, pa, v);
        const Split a = split8(v);
        // the smallest products first; FN sums apart, so none waits for the last
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j].h, a.l, acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j].l, a.h, acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j].m, a.m, acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j].h, a.m, acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j].m, a.h, acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma32(b[j].h, a.h, acc[i][j]);
    }
}
// The same tile's products of 16 rows from wm on, in fp32.
template <typename TA, typename TB, int FN>
__device__ __forceinline__ void fp32_tile(const LdsChar *at, const LdsChar *bt, int wm, int wn, int pa, int pb,
                                          f32x4 (&acc)[FN]) {
    float v[8], b[8];
    TA::floats(at, wm, pa, v);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        TB::floats(bt, wn + j * 16, pb, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[j] = mfma16(b[e], v[e], acc[j]);
    }
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }
// Scales a wave's sums back and tells whether all are finite.
template <int FM, int FN>
__device__ __forceinline__ bool unscale(f32x4 (&acc)[FM][FN]) {
    bool fine = true;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                fine = fine && finite(acc[i][j][e]);
                acc[i][j][e] *= kUnsplit;
            }
    return fine;
}
// Whether `yes` holds in any of a block's W waves; `at`: LDS that is free.
template <int W>
__device__ __forceinline__ bool any_wave(char *at, int t, bool yes) {
    int *flags = reinterpret_cast<int *>(at);
    const bool any = __builtin_amdgcn_ballot_w64(yes) != 0;
    if ((t & 63) == 0) flags[t >> 6] = any;
    __syncthreads();
    int got = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) got |= flags[i];
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(got) != 0;
}
// Of 16 rows' sums, those that are not finite, from fp32's.
template <int FN>
__device__ __forceinline__ void mend(f32x4 (&acc)[FN], const f32x4 (&fp32)[FN]) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = finite(acc[j][e]) ? acc[j][e] : fp32[j][e];
}
template <int FM, int FN>
__device__ __forceinline__ void clear(f32x4 (&acc)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
}

// What a run of E results of row m adds or needs from memory: fetched ahead of
// the sums.
template <typename T, int E>
struct Extra {
    Vec<T, E> res;
    float bias_row;
};
template <typename T, int E>
__device__ __forceinline__ void extra_fetch(const OpsGemmArgs &g, int64_t m, int64_t n, Extra<T, E> &x) {
    if (m >= g.m || n >= g.n) return;
    if (g.res) x.res = load_upto<T, E>(static_cast<const T *>(g.res) + m * g.ldr + n, g.n - n);
    if (g.bias && g.bias_rows) x.bias_row = param<T>(g.bias, m, g.bias_f32);
}
// The bias of columns n on, zeros where it runs along the rows.
template <typename T, int E>
__device__ __forceinline__ void bias_fetch(const OpsGemmArgs &g, int64_t n, float *bias) {
#pragma unroll
    for (int e = 0; e < E; ++e) bias[e] = g.bias && !g.bias_rows && n + e < g.n ? param<T>(g.bias, n + e, g.bias_f32) : 0.0f;
}
// Bias, z, activation and residual for E consecutive n of row m, rounding once
// to T at each store. The sum and all of this are fp32.
template <typename T, int E>
__device__ __forceinline__ void gemm_finish(const OpsGemmArgs &g, int64_t m, int64_t n, float *v, const float *bias,
                                            const Extra<T, E> &x) {
    if (m >= g.m || n >= g.n) return;
    const int64_t have = g.n - n;
    if (g.bias) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += g.bias_rows ? x.bias_row : bias[e];
    }
    Vec<T, E> o;
    if (g.z) {
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(v[e]);
        store_upto<T, E>(static_cast<T *>(g.z) + m * g.ldz + n, o, have);
    }
    act_fwd_n<E>(g.act, g.slope, v);
    if (g.res) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += to_f<T>(x.res.v[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(v[e]);
    store_upto<T, E>(static_cast<T *>(g.c) + m * g.ldc + n, o, have);
}

// Which tile and split a block takes. Consecutive blocks go to the 8 XCDs in
// turn, each with an L2 of its own: ids are dealt so that an XCD walks one
// contiguous run, and the run goes up 8 tiles of m before it moves along n,
// so the tiles under one L2 share operands.
__device__ __forceinline__ void gemm_place(const OpsGemmArgs &g, int &tm, int &tn, int &s) {
    const int n = gridDim.x, id = blockIdx.x, x = id & 7, q = n >> 3, r = n & 7;
    int nid = x * q + min(x, r) + (id >> 3);
    const int tiles = g.tiles_m * g.tiles_n;
    s = nid / tiles;
    nid -= s * tiles;
    const int band = nid / (8 * g.tiles_n), m0 = band * 8, h = min(8, g.tiles_m - m0);
    nid -= band * 8 * g.tiles_n;
    tn = nid / h;
    tm = m0 + nid - tn * h;
}

// A wave's FM x FN blocks of 16 x 16 from (m0, n0) on: finished, or as split
// s's partial sums. 32 rows at a time go through the wave's own part of LDS
// (`at`, gemm_write_bytes<FN>() of it), rows four floats longer than they are
// so that 16 rows' writes fall into different banks; what comes back is 16
// bytes of results a lane, whole lines of C a wave, with the bias of a lane's
// columns held in registers and the residual on its way before the sums.
// (Written from the accumulators, with a bias load each, a 256 x 256 tile's
// 32 quads a lane took 49 us.)
template <int FN>
constexpr int gemm_write_bytes() {
    return 32 * (FN * 16 + 4) * 4;
}
template <typename T, int FM, int FN>
__device__ __forceinline__ void gemm_write(const OpsGemmArgs &g, int64_t m0, int64_t n0, int s, int l, char *at,
                                           const f32x4 (&acc)[FM][FN]) {
    constexpr int E = 16 / sizeof(T), LD = FN * 16 + 4, LANES = FN * 16 / E, ROWS = 64 / LANES, STEPS = 32 / ROWS;
    static_assert(FM % 2 == 0 && LANES <= 64, "");
    float *own = reinterpret_cast<float *>(at);
    const int lr = l / LANES, lc = l % LANES * E;
    const int64_t n = n0 + lc;
    float bias[E];
    if (g.splits == 1) bias_fetch<T, E>(g, n, bias);
#pragma unroll
    for (int i = 0; i < FM; i += 2) {
        const int64_t m = m0 + i * 16 + lr;
        Extra<T, E> x[STEPS];
        if (g.splits == 1 && (g.res || g.bias_rows)) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k) extra_fetch<T, E>(g, m + k * ROWS, n, x[k]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                *reinterpret_cast<f32x4 *>(own + (h * 16 + (l & 15)) * LD + j * 16 + (l >> 4) * 4) = acc[i + h][j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            float v[E];
            const float *p = own + (k * ROWS + lr) * LD + lc;
#pragma unroll
            for (int e = 0; e < E; e += 4) *reinterpret_cast<f32x4 *>(v + e) = *reinterpret_cast<const f32x4 *>(p + e);
            if (g.splits == 1) {
                gemm_finish<T, E>(g, m + k * ROWS, n, v, bias, x[k]);
            } else if (m + k * ROWS < g.m && n < g.n) {
                Vec<float, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = v[e];
                store_upto<float, E>(g.part + ((int64_t)s * g.m + m + k * ROWS) * g.n + n, o, g.n - n);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// WM x WN waves of 64 lanes, each (BM / WM) x (BN / WN) of the tile.
template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BK_>
__device__ __forceinline__ void gemm_tile(const OpsGemmArgs &g, char *lds) {
    constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Tile<T, AK, BM, NT> TA;
    typedef Tile<T, BK_, BN, NT> TB;
    constexpr int BK = TA::BK, ABYTES = BM * 128, STAGE = (BM + BN) * 128;
    int tm, tn, s;
    gemm_place(g, tm, tn, s);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int kbeg = s * g.kchunk, kend = min(g.k, kbeg + g.kchunk);
    const int t = threadIdx.x, l = t & 63, w = t >> 6, wm = w / WN * (BM / WM), wn = w % WN * (BN / WN);
    const int rows_a = min((int64_t)BM, g.m - m0), rows_b = min((int64_t)BN, g.n - n0);
    const T *ga = static_cast<const T *>(g.a) + (AK ? m0 * g.lda + kbeg : kbeg * g.lda + m0);
    const T *gb = static_cast<const T *>(g.b) + (BK_ ? n0 * g.ldb + kbeg : kbeg * g.ldb + n0);
    typename TA::Chunk ra[TA::PER];
    typename TB::Chunk rb[TB::PER];
    auto fetch = [&](int k0) {
        TA::fetch(ra, ga + (AK ? k0 : k0 * g.lda), g.lda, t, rows_a, kend - kbeg - k0);
        TB::fetch(rb, gb + (BK_ ? k0 : k0 * g.ldb), g.ldb, t, rows_b, kend - kbeg - k0);
    };
    auto put = [&](char *at) {
#pragma unroll
        for (int i = 0; i < TA::PER; ++i) *reinterpret_cast<u32x4 *>(at + (i * NT + t) * 16) = __builtin_bit_cast(u32x4, ra[i]);
#pragma unroll
        for (int i = 0; i < TB::PER; ++i)
            *reinterpret_cast<u32x4 *>(at + ABYTES + (i * NT + t) * 16) = __builtin_bit_cast(u32x4, rb[i]);
    };
    f32x4 acc[FM][FN];
    const int nk = (kend - kbeg + BK - 1) / BK, pa = TA::lane_part(l), pb = TB::lane_part(l);
    auto run = [&](auto compute) {
        if (nk > 0) {
            fetch(0);
            put(lds);
        }
        __syncthreads();
        for (int kt = 0; kt < nk; ++kt) {
            if (kt + 1 < nk) fetch((kt + 1) * BK);
            const LdsChar *at = (LdsChar *)lds + (kt & 1) * STAGE;
            compute(at, at + ABYTES);
            if (kt + 1 < nk) put(lds + ((kt + 1) & 1) * STAGE);
            __syncthreads();
        }
    };
    clear(acc);
    run([&](const LdsChar *at, const LdsChar *bt) {
        if constexpr (sizeof(T) == 4) {
            split_tile<TA, TB, FM, FN>(at, bt, wm, wn, pa, pb, acc);
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                typename Mma<T>::Frag fa[FM], fb[FN];
#pragma unroll
                for (int i = 0; i < FM; ++i) fa[i] = TA::frag(at, wm + i * 16, kk, pa);
#pragma unroll
                for (int j = 0; j < FN; ++j) fb[j] = TB::frag(bt, wn + j * 16, kk, pb);
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::go(fb[j], fa[i], acc[i][j]);
            }
        }
    });
    if constexpr (sizeof(T) == 4) {
        // sums that are not finite, of operands too large or not finite
        // themselves, are formed again in fp32: 16 of a wave's rows at a time,
        // the others keep their bits
        if (any_wave<WM * WN>(lds, t, !unscale(acc)))
            for (int h = 0; h < FM; ++h) {
                f32x4 again[1][FN];
                clear(again);
                run([&](const LdsChar *at, const LdsChar *bt) {
                    fp32_tile<TA, TB, FN>(at, bt, wm + h * 16, wn, pa, pb, again[0]);
                });
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    if (i == h) mend(acc[i], again[0]);
            }
    }
    // behind the loop's last barrier: no wave reads the tiles any more
    gemm_write<T, FM, FN>(g, m0 + wm, n0 + wn, s, l, lds + w * gemm_write_bytes<FN>(), acc);
}

// The splits' sums added in a fixed order, then the epilogue: WAYS threads to
// four results, each every WAYS-th split, joined through LDS.
template <typename T, int WAYS>
__device__ __forceinline__ void gemm_join(const OpsGemmArgs &g) {
    constexpr int Q = 256 / WAYS;
    __shared__ f32x4 sh[WAYS > 1 ? 256 : 1];
    const int64_t quads = ((int64_t)g.n + 3) / 4, total = quads * g.m, plane = (int64_t)g.m * g.n;
    const int q = threadIdx.x % Q, way = threadIdx.x / Q;
    for (int64_t i0 = (int64_t)blockIdx.x * Q; i0 < total; i0 += (int64_t)gridDim.x * Q) {
        const int64_t i = i0 + q, m = i / quads, n = (i - m * quads) * 4;
        f32x4 v = {0, 0, 0, 0};
        if (i < total) {
            const float *p = g.part + m * g.n + n;
#pragma unroll 4
            for (int s = way; s < g.splits; s += WAYS) {
                const Vec<float, 4> o = load_upto<float, 4>(p + s * plane, g.n - n);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += o.v[e];
            }
        }
        if constexpr (WAYS > 1) {
            __syncthreads();
            sh[threadIdx.x] = v;
            __syncthreads();
            if (way) continue;
#pragma unroll
            for (int k = 1; k < WAYS; ++k) v += sh[k * Q + q];
        }
        if (i >= total) continue;
        float r[4] = {v[0], v[1], v[2], v[3]}, bias[4];
        Extra<T, 4> x;
        bias_fetch<T, 4>(g, n, bias);
        extra_fetch<T, 4>(g, m, n, x);
        gemm_finish<T, 4>(g, m, n, r, bias, x);
    }
}

// Lines of any alignment to lines of whole 16 bytes, four vectors a thread.
template <typename T>
__device__ __forceinline__ void pack_lines(const OpsPackArgs &args) {
    constexpr int E = 16 / sizeof(T);
    const OpsPackJob &a = args.job[blockIdx.y];
    const int group = blockIdx.x / a.segs, seg = blockIdx.x - group * a.segs, t = threadIdx.x;
    const int64_t line = (int64_t)group * (256 >> a.shift) + (t >> a.shift);
    if (line >= a.lines) return;
    const T *src = static_cast<const T *>(a.src) + line * a.src_ld;
    T *dst = static_cast<T *>(a.dst) + line * a.dst_ld;
    const int64_t v0 = ((int64_t)seg << (a.shift + 2)) + (t & ((1 << a.shift) - 1));
    Vec<T, E> v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t at = (v0 + ((int64_t)j << a.shift)) * E;
        v[j] = load_upto<T, E>(src + at, a.extent - at);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t at = (v0 + ((int64_t)j << a.shift)) * E;
        if (at < a.dst_ld) store_n<T, E>(dst + at, v[j]);
    }
}
extern "C" __global__ __launch_bounds__(256) void mxo_pack_16(OpsPackArgs a) { pack_lines<f16>(a); }
extern "C" __global__ __launch_bounds__(256) void mxo_pack_32(OpsPackArgs a) { pack_lines<float>(a); }

#define OPS_GEMM1(name, T, BM, BN, WM, WN, tag, AK, BK)                                                    \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxo_gemm_##name##_##BM##x##BN##_##tag(      \
        OpsGemmArgs g) {                                                                                   \
        __shared__ __align__(128) char lds[2 * (BM + BN) * 128];                                           \
        gemm_tile<T, BM, BN, WM, WN, AK, BK>(g, lds);                                                      \
    }
#define OPS_GEMM(name, T, BM, BN, WM, WN)                    \
    OPS_GEMM1(name, T, BM, BN, WM, WN, kk, true, true)       \
    OPS_GEMM1(name, T, BM, BN, WM, WN, km, true, false)      \
    OPS_GEMM1(name, T, BM, BN, WM, WN, mk, false, true)      \
    OPS_GEMM1(name, T, BM, BN, WM, WN, mm, false, false)

#define OPS_GEMM_TYPE(name, T)                                                              \
    OPS_GEMM(name, T, 128, 128, 2, 2)                                                       \
    OPS_GEMM(name, T, 64, 64, 2, 2)                                                         \
    extern "C" __global__ __launch_bounds__(256) void mxo_join_##name(OpsGemmArgs g) { gemm_join<T, 1>(g); }                \
    extern "C" __global__ __launch_bounds__(256) void mxo_join8_##name(OpsGemmArgs g) { gemm_join<T, 8>(g); }

OPS_GEMM_TYPE(bf16, bf16)
OPS_GEMM_TYPE(f16, f16)
OPS_GEMM_TYPE(f32, float)
