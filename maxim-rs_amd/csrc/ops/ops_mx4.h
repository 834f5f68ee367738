// 4-bit blocks: 32 elements along k of 1 sign, 2 exponent and 1 mantissa bit
// (0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale 2^(s - 127) of 8 bits, 255 for NaN.
//
// Quantising: with m the block's largest magnitude, s - 127 = floor(log2 m) - 2
// (4, the largest element's power of two, takes m's), at least -127; elements
// are x / 2^(s - 127) rounded to nearest, ties to even, and 6 at most. The
// quotient is exact, so one rounding is all. A block with a NaN or an infinity
// is NaN throughout.
#pragma once

#include "mx4_args.h"
#include "ops_gemm_big.h"

typedef int i32x8 __attribute__((ext_vector_type(8)));

// The scale of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// 2^-(s - 127), by which elements are multiplied (exactly); 0 for NaN blocks.
__device__ __forceinline__ float mx4_inverse(uint32_t s) {
    return s == 255 ? 0.0f : __builtin_bit_cast(float, (254 - s) << 23);
}
__device__ __forceinline__ float mx4_power(uint32_t s) {
    return __builtin_bit_cast(float, s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
// Eight values, already divided, as four bytes of codes, the first in the
// lowest bits.
__device__ __forceinline__ uint32_t mx4_codes(const float *v, float inverse) {
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __builtin_amdgcn_fmed3f(v[e] * inverse, -6.0f, 6.0f);
    uint32_t u = 0;
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[0], q[1], 1.0f, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[2], q[3], 1.0f, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[4], q[5], 1.0f, 2);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, q[6], q[7], 1.0f, 3);
    return u;
}
// Eight codes' values, of which the first four have one scale and the others
// another.
__device__ __forceinline__ void mx4_values(uint32_t u, float scale, float scale2, float *v) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#define OPS_MX4_PAIR(i)                                                         \
    {                                                                           \
        const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, i);   \
        v[2 * i] = p[0] * (i < 2 ? scale : scale2), v[2 * i + 1] = p[1] * (i < 2 ? scale : scale2); \
    }
    OPS_MX4_PAIR(0) OPS_MX4_PAIR(1) OPS_MX4_PAIR(2) OPS_MX4_PAIR(3)
#undef OPS_MX4_PAIR
}
// A scale's place in its group and tile: line r of 64, block b of 8.
__device__ __forceinline__ int scale_at(int r, int b) { return (b & 3) * 128 + (r & 15) * 8 + (r >> 4) * 2 + (b >> 2); }

// Rows with contiguous features: a block takes 32 rows (half a group) by a
// tile, 32 lanes a row with eight elements each, four lanes a block of 32. Bound
// by memory: 8192 x 4096 bf16, 85 MB, 18 to 20 us, 4.3 to 4.7 TB/s (64 rows a
// block, whose registers let fewer blocks onto a CU: 22 to 27).
template <typename T>
__device__ __forceinline__ void mx4_quantize_rows(const Mx4CodeArgs &a) {
    __shared__ uint32_t sh[64];
    const int t = threadIdx.x, lane = t & 31, tile = blockIdx.x % a.tiles;
    const int64_t half = blockIdx.x / a.tiles, r0 = half * 32;
    const int64_t k = (int64_t)tile * 256 + lane * 8, have = a.cols - k;
    if (t < 64) sh[t] = 0;  // scales of rows that are not there
    __syncthreads();
    Vec<T, 8> x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + i * 8 + (t >> 5);
        x[i] = load_upto<T, 8>(static_cast<const T *>(a.x) + min(r, a.rows - 1) * a.rs + k, have);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (t >> 5);
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = to_f<T>(x[i].v[e]);
            top = max(top, magnitude(v[e]));
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        const uint32_t s = mx4_scale(top), u = mx4_codes(v, mx4_inverse(s));
        if (r0 + row >= a.rows) continue;
        *reinterpret_cast<uint32_t *>(a.codes + ((r0 + row) * a.tiles + tile) * 128 + lane * 4) = u;
        // a half group's scales are every other dword of its group's
        const int at = scale_at(row, lane >> 2);
        if ((lane & 3) == 0) reinterpret_cast<uint8_t *>(sh)[(at >> 3) * 4 + (at & 3)] = (uint8_t)s;
    }
    __syncthreads();
    if (t < 64) {
        uint32_t *scales = reinterpret_cast<uint32_t *>(a.scales) + ((half >> 1) * a.tiles + tile) * 128 + t * 2;
        scales[half & 1] = sh[t];
        if (!(half & 1) && r0 + 32 >= a.rows) scales[1] = 0;  // a half group that no block has
    }
}

// Planar order: a block takes 64 positions (fp32) or 128 by a tile, a lane one
// or two positions (4 bytes of a feature's plane) of two of the tile's eight
// blocks. The codes go to memory through LDS, whole lines at a time. 176 planes
// of 137728 bf16 positions, 66 MB, 18 us, and back 20 (one position a lane,
// straight to memory: 73 in all); 100 planes of 65536 fp32, 35 MB, 9.8 and 7-8.
template <typename T>
__device__ __forceinline__ void mx4_quantize_planar(const Mx4CodeArgs &a, char *codes, uint32_t *sh) {
    constexpr int N = 4 / sizeof(T), ROWS = 64 * N;
    const int t = threadIdx.x, l = t & 63, w = t >> 6, tile = blockIdx.x % a.tiles;
    const int64_t part = blockIdx.x / a.tiles, r0 = part * ROWS, r = r0 + l * N;
    const int64_t have = a.rows - r;
    for (int b = w; b < 8; b += 4) {
        const int64_t k = (int64_t)tile * 256 + b * 32;
        Vec<T, N> x[32];
        const T *p = static_cast<const T *>(a.x) + r * a.rs + k * a.cs;
        if (k + 32 <= a.cols && have >= N) {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = load_n<T, N>(p + e * a.cs);
        } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = load_upto<T, N>(p + e * a.cs, k + e < a.cols ? have : 0);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[32];
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                v[e] = to_f<T>(x[e].v[i]);
                top = max(top, magnitude(v[e]));
            }
            const uint32_t s = mx4_scale(top);
            const float inverse = mx4_inverse(s);
            u32x4 u;
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = mx4_codes(v + 8 * j, inverse);
            const int row = l * N + i;
            *reinterpret_cast<u32x4 *>(codes + row * 128 + ((b ^ (l & 7)) << 4)) = u;
            reinterpret_cast<uint8_t *>(sh)[(row >> 6) * 512 + scale_at(row & 63, b)] = (uint8_t)s;
        }
    }
    __syncthreads();
    // eight lanes a line
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i) {
        const int row = i * 32 + (t >> 3), c = t & 7;
        if (r0 + row < a.rows)
            *reinterpret_cast<u32x4 *>(a.codes + ((r0 + row) * a.tiles + tile) * 128 + c * 16) =
                *reinterpret_cast<const u32x4 *>(codes + row * 128 + ((c ^ (row / N & 7)) << 4));
    }
    // the groups that have rows
    for (int i = t; i < 128 * N; i += 256) {
        const int64_t group = part * N + i / 128;
        if (group * 64 < a.rows) reinterpret_cast<uint32_t *>(a.scales)[(group * a.tiles + tile) * 128 + i % 128] = sh[i];
    }
}

// And back, by the same blocks; all of a block's codes are on their way before
// the first is used (one by one 23.5 us for 8192 x 4096 bf16, so 15.2, 5.6 TB/s).
template <typename T>
__device__ __forceinline__ void mx4_dequantize_rows(const Mx4CodeArgs &a) {
    const int t = threadIdx.x, lane = t & 31, tile = blockIdx.x % a.tiles;
    const int64_t group = blockIdx.x / a.tiles, r0 = group * 64;
    const uint8_t *scales = a.scales + (group * a.tiles + tile) * 512;
    // fp32: a lane's eight elements are four of each half, so that a row's
    // stores lie side by side
    constexpr bool WIDE = sizeof(T) == 4;
    uint32_t u[8];
    uint8_t s[8], s2[8];
    // (rows past the last are the last again)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = (int)min((int64_t)(i * 8 + (t >> 5)), a.rows - 1 - r0);
        const uint8_t *line = a.codes + ((r0 + row) * a.tiles + tile) * 128;
        if (WIDE) {
            u[i] = *reinterpret_cast<const uint16_t *>(line + lane * 2) |
                   (uint32_t) * reinterpret_cast<const uint16_t *>(line + 64 + lane * 2) << 16;
            s[i] = scales[scale_at(row, lane >> 3)];
            s2[i] = scales[scale_at(row, 4 + (lane >> 3))];
        } else {
            u[i] = *reinterpret_cast<const uint32_t *>(line + lane * 4);
            s[i] = s2[i] = scales[scale_at(row, lane >> 2)];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + i * 8 + (t >> 5);
        if (r >= a.rows) return;
        float v[8];
        mx4_values(u[i], mx4_power(s[i]), mx4_power(s2[i]), v);
        T *y = static_cast<T *>(a.y) + r * a.rs;
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) {
            const int64_t k = (int64_t)tile * 256 + h * 128 + lane * E;
            Vec<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.v[e] = from_f<T>(v[h * E + e]);
            if (k < a.cols) store_out<T, E>(y + k, o, a.cols - k);
        }
    }
}
template <typename T>
__device__ __forceinline__ void mx4_dequantize_planar(const Mx4CodeArgs &a, char *codes, uint32_t *sh) {
    constexpr int N = 4 / sizeof(T), ROWS = 64 * N;
    const int t = threadIdx.x, l = t & 63, w = t >> 6, tile = blockIdx.x % a.tiles;
    const int64_t part = blockIdx.x / a.tiles, r0 = part * ROWS, r = r0 + l * N, have = a.rows - r;
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i) {
        const int row = i * 32 + (t >> 3), c = t & 7;
        const int64_t from = min(r0 + row, a.rows - 1);
        *reinterpret_cast<u32x4 *>(codes + row * 128 + ((c ^ (row / N & 7)) << 4)) =
            *reinterpret_cast<const u32x4 *>(a.codes + (from * a.tiles + tile) * 128 + c * 16);
    }
    for (int i = t; i < 128 * N; i += 256) {
        const int64_t group = min(part * N + i / 128, (a.rows - 1) / 64);
        sh[i] = reinterpret_cast<const uint32_t *>(a.scales)[(group * a.tiles + tile) * 128 + i % 128];
    }
    __syncthreads();
    if (have <= 0) return;
    for (int b = w; b < 8; b += 4) {
        const int64_t k = (int64_t)tile * 256 + b * 32;
        if (k >= a.cols) return;
        float v[N][32];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = l * N + i;
            const u32x4 u = *reinterpret_cast<const u32x4 *>(codes + row * 128 + ((b ^ (l & 7)) << 4));
            const float scale = mx4_power(reinterpret_cast<const uint8_t *>(sh)[(row >> 6) * 512 + scale_at(row & 63, b)]);
#pragma unroll
            for (int j = 0; j < 4; ++j) mx4_values(u[j], scale, scale, v[i] + 8 * j);
        }
        T *p = static_cast<T *>(a.y) + r * a.rs + k * a.cs;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            Vec<T, N> o;
#pragma unroll
            for (int i = 0; i < N; ++i) o.v[i] = from_f<T>(v[i][e]);
            if (k + e < a.cols) store_upto<T, N>(p + e * a.cs, o, have);
        }
    }
}

// ------------------------------------------------------------- the product

// One matrix instruction: 16 x 16 sums of 128 products, of which lane l brings
// 32 of line l % 16, k's 32 (l / 16) on, with their scale in byte OB of sb
// (first operand) or OA of sa.
template <int OB, int OA>
__device__ __forceinline__ f32x4 mx4_mma(const u32x4 &b, const u32x4 &a, f32x4 c, uint32_t sb, uint32_t sa) {
    const i32x8 wb = __builtin_bit_cast(i32x8, __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1));
    const i32x8 wa = __builtin_bit_cast(i32x8, __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1));
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wb, wa, c, 4, 4, OB, (int)sb, OA, (int)sa);
}
// The same with the bytes known once loops are unrolled.
__device__ __forceinline__ f32x4 mx4_mma(int ob, int oa, const u32x4 &b, const u32x4 &a, f32x4 c, uint32_t sb,
                                         uint32_t sa) {
#define OPS_MX4_CASE(i, j) \
    case i * 4 + j: return mx4_mma<i, j>(b, a, c, sb, sa);
    switch (ob * 4 + oa) {
        OPS_MX4_CASE(0, 0) OPS_MX4_CASE(0, 1) OPS_MX4_CASE(0, 2) OPS_MX4_CASE(0, 3)
        OPS_MX4_CASE(1, 0) OPS_MX4_CASE(1, 1) OPS_MX4_CASE(1, 2) OPS_MX4_CASE(1, 3)
        OPS_MX4_CASE(2, 0) OPS_MX4_CASE(2, 1) OPS_MX4_CASE(2, 2) OPS_MX4_CASE(2, 3)
        OPS_MX4_CASE(3, 0) OPS_MX4_CASE(3, 1) OPS_MX4_CASE(3, 2)
        default: return mx4_mma<3, 3>(b, a, c, sb, sa);
    }
#undef OPS_MX4_CASE
}

// 4 bytes a lane into LDS at `at` + lane * 4.
__device__ __forceinline__ void lds_load4(__amdgpu_buffer_rsrc_t r, char *at, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)at, 4, off, 0, 0, 0);
}

// C's BM x BM tile: a tile's lines are 128 bytes as those of 16-bit operands
// are, and so are the fragments, so this is gemm_direct's 16-bit way with four
// times the k's a tile and their scales beside them in LDS. A dword of scales a
// lane serves four instructions (two fragments' both halves of k), so they cost
// three LDS reads a tile; read at the tile's start instead of a phase ahead,
// 4096^3 took 38.4 us, not 36.5. bf16 results, with x quantised: 4096^3 47 us,
// 8192^3 278 (4.0 PFLOP/s; the instructions alone reach 8.0 on random operands).
// A step of k takes 1.6 us where its products take 0.85: bound by the tiles' way
// into LDS (without memory behind it 1.23) and out of it (without products 1.06).
template <typename T, int BM, int WM, int WN, int ST>
__device__ __forceinline__ void mx4_gemm(const Mx4GemmArgs &m, const Stage (&st)[ST], char *const (&sc)[ST]) {
    static_assert((WM * WN + 3) / 4 * gemm_write_bytes<BM / WN / 16>() <= BM * 128, "");
    constexpr int NT = 64 * WM * WN, FM = BM / WM / 16, FN = BM / WN / 16, W = WM * WN;
    typedef Tile<bf16, true, BM, NT> TT;
    const OpsGemmArgs &g = m.g;
    int tm, tn, s;
    gemm_place(g, tm, tn, s);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BM;
    const int kbeg = s * g.kchunk, kend = min(g.k, kbeg + g.kchunk), nk = kend - kbeg;
    const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = w / WN * (BM / WM), wn = w % WN * (BM / WN);
    const int rows_a = min((int64_t)BM, g.m - m0), rows_b = min((int64_t)BM, g.n - n0);
    const int ld = g.k * 128;
    int r, k;
    TT::where(t, r, k);
    const uint32_t off = r * ld + k * 2;
    const char *next_a = reinterpret_cast<const char *>(m.a) + m0 * ld + kbeg * 128;
    const char *next_b = reinterpret_cast<const char *>(m.b) + n0 * ld + kbeg * 128;
    // Scales: 256 bytes a wave and operand, or (64 x 64 tiles) the first two
    // waves A's and the others B's; the lines of groups past the last are not
    // there.
    constexpr int GROUPS = BM / 64, SL = GROUPS * 2 == W ? 2 : 1;
    static_assert(GROUPS * 2 == W || (GROUPS == 1 && W == 4), "");
    const int sg = SL == 2 ? w >> 1 : 0, sh = w & 1;
    const int64_t groups_a = (g.m + 63) / 64, groups_b = (g.n + 63) / 64;
    const int ga = min((int64_t)GROUPS, groups_a - m0 / 64), gb = min((int64_t)GROUPS, groups_b - n0 / 64);
    const int lds_ = g.k * 512;
    const uint32_t soff = sg * lds_ + sh * 256 + l * 4;
    const char *next_sa = reinterpret_cast<const char *>(m.sa) + m0 / 64 * lds_ + (int64_t)kbeg * 512;
    const char *next_sb = reinterpret_cast<const char *>(m.sb) + n0 / 64 * lds_ + (int64_t)kbeg * 512;
    int left = nk;
    auto stage = [&](const Stage &to, char *scales) {
        const bool live = __builtin_amdgcn_readfirstlane(left) > 0;
        auto buffer = [&](const char *p, int bytes) {
            return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, live ? bytes : 0, 0x00020000);
        };
        const __amdgpu_buffer_rsrc_t ba = buffer(next_a, rows_a * ld), bb = buffer(next_b, rows_b * ld);
#pragma unroll
        for (int i = 0; i < TT::PER; ++i) lds_load16(ba, to.a + (i * NT + w * 64) * 16, off + i * (NT / 8) * ld);
#pragma unroll
        for (int i = 0; i < TT::PER; ++i) lds_load16(bb, to.b + (i * NT + w * 64) * 16, off + i * (NT / 8) * ld);
        if constexpr (SL == 2) {
            lds_load4(buffer(next_sa, ga * lds_), scales + w * 256, soff);
            lds_load4(buffer(next_sb, gb * lds_), scales + GROUPS * 512 + w * 256, soff);
        } else {
            lds_load4(w < 2 ? buffer(next_sa, ga * lds_) : buffer(next_sb, gb * lds_), scales + w * 256, soff);
        }
        next_a += 128, next_b += 128, next_sa += 512, next_sb += 512;
        --left;
    };
    f32x4 acc[FM][FN];
    clear(acc);
    constexpr int LOADS = 2 * TT::PER + SL, AHEAD = (ST - 2) * LOADS;
    const int part = TT::lane_part(l);
    constexpr int HM = FM / 2;
    u32x4 fa[2][HM], fb[2][FN];
    // a tile's scales, and the next one's: a dword has two fragments' bytes of
    // both halves of k
    uint32_t xa[FM / 2], xb[FN / 2], ya[FM / 2], yb[FN / 2];
    auto take = [&](const LdsChar *at, int base, int kk) {
        return __builtin_bit_cast(u32x4, TT::frag(at, base, kk, part));
    };
    auto take_a = [&](const Stage &c, int kk, int h) {
#pragma unroll
        for (int i = 0; i < HM; ++i) fa[h][i] = take((LdsChar *)c.a, wm + (h * HM + i) * 16, kk);
    };
    auto take_b = [&](const Stage &c, int kk) {
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[kk][j] = take((LdsChar *)c.b, wn + j * 16, kk);
    };
    auto take_scales = [&](const char *scales) {
        typedef const __attribute__((address_space(3))) uint32_t *SP;
        const LdsChar *pa = (LdsChar *)scales + wm / 64 * 512 + (wm & 32) / 8 + l * 8;
        const LdsChar *pb = (LdsChar *)scales + GROUPS * 512 + wn / 64 * 512 + (wn & 32) / 8 + l * 8;
#pragma unroll
        for (int i = 0; i < FM / 2; ++i) ya[i] = *(SP)(pa + i / 2 * 512 + i % 2 * 4);
#pragma unroll
        for (int j = 0; j < FN / 2; ++j) yb[j] = *(SP)(pb + j / 2 * 512 + j % 2 * 4);
    };
    auto next_scales = [&] {
#pragma unroll
        for (int i = 0; i < FM / 2; ++i) xa[i] = ya[i];
#pragma unroll
        for (int j = 0; j < FN / 2; ++j) xb[j] = yb[j];
    };
    auto multiply = [&](int kk, int h) {
#pragma unroll
        for (int i = 0; i < HM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int f = h * HM + i;
                acc[f][j] = mx4_mma(j % 2 * 2 + kk, f % 2 * 2 + kk, fb[kk][j], fa[h][i], acc[f][j], xb[j / 2], xa[f / 2]);
            }
    };
    // gemm_direct's four phases; the next tile's scales are read as soon as it is
    // there.
    auto tile = [&](const Stage &c, const Stage &n, char *csc, const char *nsc) {
        constexpr int MP = HM * FN;
        take_a(c, 0, 1);
        multiply(0, 0);
        spread<HM, MP>();
        take_b(c, 1);
        take_a(c, 1, 0);
        multiply(0, 1);
        spread<HM + FN, MP>();
        take_a(c, 1, 1);
        multiply(1, 0);
        spread<HM, MP>();
        tiles_landed<AHEAD>();
        take_scales(nsc);
        stage(c, csc);
        __builtin_amdgcn_sched_barrier(0);
        take_b(n, 0);
        take_a(n, 0, 0);
        multiply(1, 1);
        spread<HM + FN, MP>();
        next_scales();
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) stage(st[i], sc[i]);
    tiles_landed<AHEAD + LOADS>();
    take_b(st[0], 0);
    take_a(st[0], 0, 0);
    take_scales(sc[0]);
    next_scales();
    for (int kt = 0; kt < nk; kt += ST) {
#pragma unroll
        for (int i = 0; i < ST; ++i) tile(st[i], st[(i + 1) % ST], sc[i], sc[(i + 1) % ST]);
    }
    tiles_landed<0>();
    char *own = (w & 1 ? w & 2 ? st[1].b : st[1].a : w & 2 ? st[0].b : st[0].a) + (w >> 2) * gemm_write_bytes<FN>();
    gemm_write<T, FM, FN>(g, m0 + wm, n0 + wn, s, l, own, acc);
}

// Up to 16 rows: ops_skinny.h's way, x taken to 4 bits as it is read. A lane's
// part of a fragment is one block of 32 of its row, so the block's scale needs
// no other lane. 1 x 4096 to 4096 columns, 9 MB of weights, 6.5 us in a graph of
// calls, 16 rows 9.0 (without loads ahead 7.6 and 9.3): latency of two tiles a
// wave and a launch; where k is long, mx4_plan (exec/mx4.cpp) takes the tiles.
template <typename T>
__device__ __forceinline__ void mx4_skinny(const Mx4GemmArgs &m) {
    constexpr int W = 8;
    __shared__ f32x4 sums[W][64];
    const OpsGemmArgs &g = m.g;
    const int t = threadIdx.x, l = t & 63, w = t >> 6, r = l & 15, q = l >> 4;
    // four blocks share a group's scales: those with one XCD's L2
    const int per = gridDim.x / 8, id = blockIdx.x < per * 8 ? blockIdx.x % 8 * per + blockIdx.x / 8 : blockIdx.x;
    const int64_t n0 = (int64_t)id * 16, line = min(n0 + r, (int64_t)g.n - 1);
    const int tiles = g.k, each = (tiles + W - 1) / W, kend = min(tiles, (w + 1) * each);
    const uint8_t *b = m.b + line * tiles * 128 + q * 16;
    const uint8_t *sb = m.sb + n0 / 64 * tiles * 512 + q * 128 + r * 8 + (n0 / 16 & 3) * 2;
    const T *x = reinterpret_cast<const T *>(m.a) + (int64_t)min(r, g.m - 1) * g.lda;
    f32x4 acc = {0, 0, 0, 0};
    // A tile's loads, two tiles ahead of its products (in fp32 one: x's two would
    // not fit the registers).
    constexpr int AHEAD = sizeof(T) == 2 ? 2 : 1;
    struct In {
        u32x4 b[2];
        uint32_t s;
        Vec<T, 8> x[2][4];
    };
    auto fetch = [&](int k, In &in) {
#pragma unroll
        for (int h = 0; h < 2; ++h) in.b[h] = *reinterpret_cast<const u32x4 *>(b + (int64_t)k * 128 + h * 64);
        in.s = *reinterpret_cast<const uint16_t *>(sb + (int64_t)k * 512);
        const int64_t at = (int64_t)k * 256 + q * 32;
        if ((int64_t)(k + 1) * 256 <= m.cols) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) in.x[h][i] = load_n<T, 8>(x + at + h * 128 + i * 8);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) in.x[h][i] = load_upto<T, 8>(x + at + h * 128 + i * 8, m.cols - at - h * 128 - i * 8);
        }
    };
    auto use = [&](const In &in) {
        u32x4 a[2];
        uint32_t sa[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t top = 0;
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                f[e] = to_f<T>(in.x[h][e / 8].v[e % 8]);
                top = max(top, magnitude(f[e]));
            }
            sa[h] = mx4_scale(top);
            const float inverse = mx4_inverse(sa[h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[h][i] = mx4_codes(f + 8 * i, inverse);
        }
        acc = mx4_mma<0, 0>(in.b[0], a[0], acc, in.s, sa[0]);
        acc = mx4_mma<1, 0>(in.b[1], a[1], acc, in.s, sa[1]);
    };
    In in[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (w * each + i < kend) fetch(w * each + i, in[i]);
    for (int k = w * each; k < kend; k += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (k + i < kend) use(in[i]);
            if (k + i + AHEAD < kend) fetch(k + i + AHEAD, in[i]);
        }
    }
    sums[w][l] = acc;
    __syncthreads();
    if (t >= 64) return;
    f32x4 v = sums[0][l];
#pragma unroll
    for (int k = 1; k < W; ++k) v += sums[k][l];
    const int64_t row = r, n = n0 + q * 4;
    float out[4] = {v[0], v[1], v[2], v[3]}, bias[4];
    Extra<T, 4> e;
    bias_fetch<T, 4>(g, n, bias);
    extra_fetch<T, 4>(g, row, n, e);
    gemm_finish<T, 4>(g, row, n, out, bias, e);
}
