// Products of aligned 16-bit operands: both tiles go from memory straight to
// LDS.
#pragma once

#include "ops_gemm.h"

// 16 bytes a lane from the buffer into LDS at `at` + lane * 16 (a wave's own
// 1 KiB). A lane whose offset is past the buffer's end writes zeros.
__device__ __forceinline__ void lds_load16(__amdgpu_buffer_rsrc_t r, char *at, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)at, 16, off, 0, 0, 0);
}
constexpr uint32_t kNowhere = 0x80000000u;

template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BK_>
__device__ __forceinline__ void gemm_direct(const OpsGemmArgs &g, char *a0, char *b0, char *a1, char *b1) {
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
    uint32_t oa[TA::PER], ob[TB::PER];
    int ka[TA::PER], kb[TB::PER];
#pragma unroll
    for (int i = 0; i < TA::PER; ++i) {
        int row, k;
        TA::where(i * NT + t, row, k);
        ka[i] = k;
        oa[i] = row < rows_a ? (uint32_t)(AK ? row * g.lda + k : k * g.lda + row) * sizeof(T) : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < TB::PER; ++i) {
        int row, k;
        TB::where(i * NT + t, row, k);
        kb[i] = k;
        ob[i] = row < rows_b ? (uint32_t)(BK_ ? row * g.ldb + k : k * g.ldb + row) * sizeof(T) : kNowhere;
    }
    auto stage = [&](int kt, char *at, char *bt) {
        const int k0 = kt * BK, left = kend - kbeg - k0;
        const __amdgpu_buffer_rsrc_t bufa =
            __builtin_amdgcn_make_buffer_rsrc((void *)(ga + (AK ? (int64_t)k0 : k0 * g.lda)), 0, 0x7fffffff, 0x00020000);
        const __amdgpu_buffer_rsrc_t bufb =
            __builtin_amdgcn_make_buffer_rsrc((void *)(gb + (BK_ ? (int64_t)k0 : k0 * g.ldb)), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < TA::PER; ++i) lds_load16(bufa, at + (i * NT + w * 64) * 16, ka[i] < left ? oa[i] : kNowhere);
#pragma unroll
        for (int i = 0; i < TB::PER; ++i)
            lds_load16(bufb, bt + (i * NT + w * 64) * 16, kb[i] < left ? ob[i] : kNowhere);
    };
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    auto compute = [&](const LdsChar *at, const LdsChar *bt) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            typename Mma<T>::Frag fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = TA::frag(at, wm + i * 16, kk, l);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = TB::frag(bt, wn + j * 16, kk, l);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::go(fb[j], fa[i], acc[i][j]);
        }
    };
    const int nk = (kend - kbeg + BK - 1) / BK;
    if (nk > 0) stage(0, a0, b0);
    for (int kt = 0; kt < nk; kt += 2) {
        __syncthreads();
        if (kt + 1 < nk) stage(kt + 1, a1, b1);
        compute((LdsChar *)a0, (LdsChar *)b0);
        __syncthreads();
        if (kt + 1 < nk) {
            if (kt + 2 < nk) stage(kt + 2, a0, b0);
            compute((LdsChar *)a1, (LdsChar *)b1);
        }
    }
    gemm_write<T, FM, FN>(g, m0 + wm, n0 + wn, s, l, acc);
}

#define OPS_DIRECT1(name, T, BM, BN, WM, WN, tag, AK, BK)                                                  \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxo_gemm_##name##_##BM##x##BN##_##tag##_d(  \
        OpsGemmArgs g) {                                                                                   \
        __shared__ __align__(1024) char a0[BM * 128];                                                      \
        __shared__ __align__(1024) char b0[BN * 128];                                                      \
        __shared__ __align__(1024) char a1[BM * 128];                                                      \
        __shared__ __align__(1024) char b1[BN * 128];                                                      \
        gemm_direct<T, BM, BN, WM, WN, AK, BK>(g, a0, b0, a1, b1);                                         \
    }
#define OPS_DIRECT(name, T, BM, BN, WM, WN)                    \
    OPS_DIRECT1(name, T, BM, BN, WM, WN, kk, true, true)       \
    OPS_DIRECT1(name, T, BM, BN, WM, WN, km, true, false)      \
    OPS_DIRECT1(name, T, BM, BN, WM, WN, mk, false, true)      \
    OPS_DIRECT1(name, T, BM, BN, WM, WN, mm, false, false)

OPS_DIRECT(bf16, bf16, 256, 256, 2, 4)
OPS_DIRECT(f16, f16, 256, 256, 2, 4)
OPS_DIRECT(bf16, bf16, 128, 128, 2, 2)
OPS_DIRECT(f16, f16, 128, 128, 2, 2)
