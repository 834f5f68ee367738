// Products of operands aligned to 16 bytes: both tiles go from memory straight
// to LDS.
//
// Bound by the matrix cores where there are tiles enough, at the clock their
// power leaves: bf16 8192^3 in 820-910 us (1.2-1.3 PFLOP/s; the library's
// product 680-810), 4096^3 in 108-125 us (89-100). 8192 x 2048 x 8192 with 134
// MB of results 262 us, with gelu 269, with the 134 MB of z as well 290: a
// 256 x 256 tile takes 128 KiB of a CU's 160 KiB of LDS, so no second one fits
// beside it and its results are written before its CU's next tile is begun. Two
// smaller tiles a CU hide that, and lose more in products an LDS byte read.
#pragma once

#include "ops_gemm.h"

// 16 bytes a lane from the buffer into LDS at `at` + lane * 16 (a wave's own
// 1 KiB). A lane whose offset is past the buffer's end writes zeros.
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t r, char *at, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)at, 16, off, 0, 0, 0);
}
constexpr uint32_t kNowhere = 0x80000000u;

// Waits for this wave's loads into LDS, all but the last `AHEAD` of them, and
// its reads from it, then for the other waves: a barrier alone waits for
// neither.
template <int AHEAD>
__device__ __forceinline__ void tiles_landed() {
    static_assert(AHEAD < 64, "");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (AHEAD & 15) | (AHEAD >> 4) << 14);  // vmcnt(AHEAD), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The order of a phase: its LDS reads, which the next phase multiplies, spread
// over its own products. (Left alone the compiler puts each read right before
// its use.)
template <int READS, int PRODUCTS>
__device__ __forceinline__ void spread() {
    constexpr int EACH = PRODUCTS / READS > 0 ? PRODUCTS / READS : 1, DONE = EACH * READS;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
        if (i * EACH < PRODUCTS) __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
    if (DONE < PRODUCTS) __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS - DONE, 0);
}

// LDS for one stage of both operands: arrays of their own, so that the compiler
// can tell a read of one stage from the loads into the others (and does not
// wait for those).
struct Stage {
    char *a, *b;
};

template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BK_, int ST>
__device__ __forceinline__ void gemm_direct(const OpsGemmArgs &g, const Stage (&st)[ST]) {
    // the epilogue takes a quarter of the waves in each of four arrays
    static_assert((WM * WN + 3) / 4 * gemm_write_bytes<BN / WN / 16>() <= BM * 128 && BM == BN, "");
    constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Tile<T, AK, BM, NT> TA;
    typedef Tile<T, BK_, BN, NT> TB;
    constexpr int BK = TA::BK;
    int tm, tn, s;
    gemm_place(g, tm, tn, s);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int kbeg = s * g.kchunk, kend = min(g.k, kbeg + g.kchunk);
    const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = w / WN * (BM / WM), wn = w % WN * (BN / WN);
    const int rows_a = min((int64_t)BM, g.m - m0), rows_b = min((int64_t)BN, g.n - n0);
    const T *ga = static_cast<const T *>(g.a) + (AK ? m0 * g.lda + kbeg : kbeg * g.lda + m0);
    const T *gb = static_cast<const T *>(g.b) + (BK_ ? n0 * g.ldb + kbeg : kbeg * g.ldb + n0);
    // A thread's chunks of a tile lie a fixed number of rows (along k: of k's)
    // apart, one offset and a step. What lies past the operand's end along the
    // strided axis is past the buffer's, past its end along the other one the
    // offset is sent there.
    // (In fp32 tiles that are contiguous along rows the swizzle differs from
    // chunk to chunk: an offset each.) All of it fits 31 bits, which the host
    // sees to (spans() in exec/ops.cpp); from tile to tile the base moves.
    constexpr int OA = AK || sizeof(T) == 2 ? 1 : TA::PER, OB = BK_ || sizeof(T) == 2 ? 1 : TB::PER;
    const int lda = (int)(g.lda * sizeof(T)), ldb = (int)(g.ldb * sizeof(T));
    const uint32_t step_a = (AK ? NT / 8 : NT / TA::CPR) * lda, step_b = (BK_ ? NT / 8 : NT / TB::CPR) * ldb;
    uint32_t oa[OA], ob[OB];
    int ka, kb;  // along k: the chunks' first k, the same in all of them
#pragma unroll
    for (int i = OA - 1; i >= 0; --i) {
        int r;
        TA::where(i * NT + t, r, ka);
        oa[i] = AK || r < rows_a ? (AK ? r * lda + ka * (int)sizeof(T) : ka * lda + r * (int)sizeof(T)) : kNowhere;
    }
#pragma unroll
    for (int i = OB - 1; i >= 0; --i) {
        int r;
        TB::where(i * NT + t, r, kb);
        ob[i] = BK_ || r < rows_b ? (BK_ ? r * ldb + kb * (int)sizeof(T) : kb * ldb + r * (int)sizeof(T)) : kNowhere;
    }
    const char *next_a = reinterpret_cast<const char *>(ga), *next_b = reinterpret_cast<const char *>(gb);
    int left = kend - kbeg;
    // the next tile, in turn
    auto stage = [&](char *at, char *bt) {
        // (the compiler clamps in the vector unit; a buffer in vector registers
        // would be loaded from lane by lane)
        const int k = __builtin_amdgcn_readfirstlane(max(0, min(left, BK)));
        const __amdgpu_buffer_rsrc_t bufa =
            __builtin_amdgcn_make_buffer_rsrc((void *)next_a, 0, (AK ? rows_a : k) * lda, 0x00020000);
        const __amdgpu_buffer_rsrc_t bufb =
            __builtin_amdgcn_make_buffer_rsrc((void *)next_b, 0, (BK_ ? rows_b : k) * ldb, 0x00020000);
        const uint32_t fa = !AK || ka < k ? oa[0] : kNowhere, fb = !BK_ || kb < k ? ob[0] : kNowhere;
#pragma unroll
        for (int i = 0; i < TA::PER; ++i)
            lds_load16(bufa, at + (i * NT + w * 64) * 16, OA > 1 ? oa[OA > 1 ? i : 0] : fa + i * step_a);
#pragma unroll
        for (int i = 0; i < TB::PER; ++i)
            lds_load16(bufb, bt + (i * NT + w * 64) * 16, OB > 1 ? ob[OB > 1 ? i : 0] : fb + i * step_b);
        next_a += AK ? 128 : BK * lda;
        next_b += BK_ ? 128 : BK * ldb;
        left -= BK;
    };
    f32x4 acc[FM][FN];
    clear(acc);
    const int nk = (kend - kbeg + BK - 1) / BK;
    constexpr int LOADS = TA::PER + TB::PER, AHEAD = (ST - 2) * LOADS;
    const int pa = TA::lane_part(l), pb = TB::lane_part(l);
    if constexpr (sizeof(T) == 4) {
        // A tile at a time: the one after the ST - 1 in LDS is sent for when
        // all waves are done with the place it takes.
        auto run = [&](auto compute) {
            next_a = reinterpret_cast<const char *>(ga), next_b = reinterpret_cast<const char *>(gb);
            left = kend - kbeg;
#pragma unroll
            for (int i = 0; i < ST - 1; ++i) stage(st[i].a, st[i].b);
            auto tile = [&](const Stage &c, const Stage &last) {
                tiles_landed<AHEAD>();
                stage(last.a, last.b);
                __builtin_amdgcn_sched_barrier(0);
                compute((LdsChar *)c.a, (LdsChar *)c.b);
            };
            int kt = 0;
            for (; kt + ST <= nk; kt += ST) {
#pragma unroll
                for (int i = 0; i < ST; ++i) tile(st[i], st[(i + ST - 1) % ST]);
            }
#pragma unroll
            for (int i = 0; i < ST - 1; ++i) {
                if (kt + i >= nk) break;
                tile(st[i], st[(i + ST - 1) % ST]);
            }
            tiles_landed<0>();
        };
        run([&](const LdsChar *at, const LdsChar *bt) { split_tile<TA, TB, FM, FN>(at, bt, wm, wn, pa, pb, acc); });
        // sums that are not finite, of operands too large or not finite
        // themselves, are formed again in fp32: 16 of a wave's rows at a time,
        // the others keep their bits
        if (any_wave<WM * WN>(st[0].a, t, !unscale(acc)))
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
    } else {
        // A tile is four phases, two halves of k by two halves of the wave's rows,
        // each multiplying fragments that the phase before it read from LDS.
        constexpr int HM = FM / 2;
        typedef typename Mma<T>::Frag Frag;
        Frag fa[2][HM], fb[2][FN];
        // In the largest tiles a fragment's address (its own register where the
        // operand is not contiguous along k) is worked out when it is read: held
        // through the loop they do not fit beside the sums.
        auto here = [&](int part) {
            if (FM * FN >= 32 && (!AK || !BK_)) asm volatile("" : "+v"(part));
            return part;
        };
        auto take_a = [&](const LdsChar *at, int kk, int h) {
            const int part = here(pa);
#pragma unroll
            for (int i = 0; i < HM; ++i) fa[h][i] = TA::frag(at, wm + (h * HM + i) * 16, kk, part);
        };
        auto take_b = [&](const LdsChar *bt, int kk) {
            const int part = here(pb);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[kk][j] = TB::frag(bt, wn + j * 16, kk, part);
        };
        auto multiply = [&](int kk, int h) {
#pragma unroll
            for (int i = 0; i < HM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[h * HM + i][j] = Mma<T>::go(fb[kk][j], fa[h][i], acc[h * HM + i][j]);
        };
        // The last phase's fragments are in registers when it begins: then, with
        // the next tile landed, the tile ST on is sent for into this one's place,
        // ST - 1 tiles' time ahead of its use. Past the last tile the loads bring
        // zeros without touching memory.
        auto tile = [&](const Stage &c, const Stage &n) {
            constexpr int RA = HM * (AK ? 1 : 2), RB = FN * (BK_ ? 1 : 2), MP = HM * FN;
            take_a((LdsChar *)c.a, 0, 1);
            multiply(0, 0);
            spread<RA, MP>();
            take_b((LdsChar *)c.b, 1);
            take_a((LdsChar *)c.a, 1, 0);
            multiply(0, 1);
            spread<RA + RB, MP>();
            take_a((LdsChar *)c.a, 1, 1);
            multiply(1, 0);
            spread<RA, MP>();
            tiles_landed<AHEAD>();
            stage(c.a, c.b);
            __builtin_amdgcn_sched_barrier(0);  // sent for here, not where the scheduler finds room
            take_b((LdsChar *)n.b, 0);
            take_a((LdsChar *)n.a, 0, 0);
            multiply(1, 1);
            spread<RA + RB, MP>();
        };
#pragma unroll
        for (int i = 0; i < ST; ++i) stage(st[i].a, st[i].b);
        tiles_landed<AHEAD + LOADS>();
        take_b((LdsChar *)st[0].b, 0);
        take_a((LdsChar *)st[0].a, 0, 0);
        // ST tiles a round and the rest one by one. (In the largest tiles, whose
        // fragments leave no registers for a second exit, the last round is filled
        // with a tile of zeros instead.)
        constexpr bool FILL = FM * FN >= 32;
        int kt = 0;
        for (; FILL ? kt < nk : kt + ST <= nk; kt += ST) {
#pragma unroll
            for (int i = 0; i < ST; ++i) tile(st[i], st[(i + 1) % ST]);
        }
        if constexpr (!FILL) {
#pragma unroll
            for (int i = 0; i < ST - 1; ++i) {
                if (kt + i >= nk) break;
                tile(st[i], st[i + 1]);
            }
        }
    }
    tiles_landed<0>();  // the last loads too, zeros: the tiles' LDS is free
    char *own = (w & 1 ? w & 2 ? st[1].b : st[1].a : w & 2 ? st[0].b : st[0].a) + (w >> 2) * gemm_write_bytes<FN>();
    gemm_write<T, FM, FN>(g, m0 + wm, n0 + wn, s, l, own, acc);
}

#define OPS_STAGE(i, BM, BN)                              \
    __shared__ __align__(1024) char a##i[BM * 128];       \
    __shared__ __align__(1024) char b##i[BN * 128];
#define OPS_DIRECT2(name, T, BM, BN, WM, WN, tag, AK, BK)                                                  \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxo_gemm_##name##_##BM##x##BN##_##tag##_d2( \
        OpsGemmArgs g) {                                                                                   \
        OPS_STAGE(0, BM, BN)                                                                               \
        OPS_STAGE(1, BM, BN)                                                                               \
        const Stage st[2] = {{a0, b0}, {a1, b1}};                                                          \
        gemm_direct<T, BM, BN, WM, WN, AK, BK, 2>(g, st);                                                  \
    }
#define OPS_DIRECT4(name, T, BM, BN, WM, WN, tag, AK, BK)                                                  \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxo_gemm_##name##_##BM##x##BN##_##tag##_d4( \
        OpsGemmArgs g) {                                                                                   \
        OPS_STAGE(0, BM, BN)                                                                               \
        OPS_STAGE(1, BM, BN)                                                                               \
        OPS_STAGE(2, BM, BN)                                                                               \
        OPS_STAGE(3, BM, BN)                                                                               \
        const Stage st[4] = {{a0, b0}, {a1, b1}, {a2, b2}, {a3, b3}};                                      \
        gemm_direct<T, BM, BN, WM, WN, AK, BK, 4>(g, st);                                                  \
    }
#define OPS_DIRECT(ST, name, T, BM, BN, WM, WN)                     \
    OPS_DIRECT##ST(name, T, BM, BN, WM, WN, kk, true, true)         \
    OPS_DIRECT##ST(name, T, BM, BN, WM, WN, km, true, false)        \
    OPS_DIRECT##ST(name, T, BM, BN, WM, WN, mk, false, true)        \
    OPS_DIRECT##ST(name, T, BM, BN, WM, WN, mm, false, false)

#define OPS_DIRECT_TYPE(name, T)              \
    OPS_DIRECT(2, name, T, 256, 256, 2, 4)    \
    OPS_DIRECT(2, name, T, 128, 128, 2, 2)    \
    OPS_DIRECT(4, name, T, 128, 128, 2, 2)    \
    OPS_DIRECT(4, name, T, 64, 64, 2, 2)

OPS_DIRECT_TYPE(bf16, bf16)
OPS_DIRECT_TYPE(f16, f16)
OPS_DIRECT(2, f32, float, 128, 128, 2, 2)
OPS_DIRECT(4, f32, float, 64, 64, 2, 2)
OPS_DIRECT(2, f32, float, 64, 64, 2, 2)
