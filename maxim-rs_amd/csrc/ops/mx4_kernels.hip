// The gfx950 code object of the 4-bit operators (include/maxim_block_ops.h).
#define OPS_GATED
#include "ops_mx4.h"

#define OPS_MX4_STAGE(i, B)                              \
    OPS_STAGE(i, B, B)                                   \
    __shared__ __align__(512) char s##i[B / 64 * 1024];
#define OPS_MX4_D2(name, T, B, WM, WN)                                                                     \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxq_gemm_##name##_##B##x##B##_d2(Mx4GemmArgs m) { \
        OPS_MX4_STAGE(0, B)                                                                                \
        OPS_MX4_STAGE(1, B)                                                                                \
        const Stage st[2] = {{a0, b0}, {a1, b1}};                                                          \
        char *const sc[2] = {s0, s1};                                                                      \
        mx4_gemm<T, B, WM, WN, 2>(m, st, sc);                                                              \
    }
#define OPS_MX4_D4(name, T, B, WM, WN)                                                                     \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void mxq_gemm_##name##_##B##x##B##_d4(Mx4GemmArgs m) { \
        OPS_MX4_STAGE(0, B)                                                                                \
        OPS_MX4_STAGE(1, B)                                                                                \
        OPS_MX4_STAGE(2, B)                                                                                \
        OPS_MX4_STAGE(3, B)                                                                                \
        const Stage st[4] = {{a0, b0}, {a1, b1}, {a2, b2}, {a3, b3}};                                      \
        char *const sc[4] = {s0, s1, s2, s3};                                                              \
        mx4_gemm<T, B, WM, WN, 4>(m, st, sc);                                                              \
    }
#define OPS_MX4_TYPE(name, T)                                                                                        \
    extern "C" __global__ __launch_bounds__(256) void mxq_quantize_rows_##name(Mx4CodeArgs a) { mx4_quantize_rows<T>(a); }     \
    extern "C" __global__ __launch_bounds__(256) void mxq_quantize_planar_##name(Mx4CodeArgs a) {                    \
        __shared__ __align__(16) char codes[64 * 4 / sizeof(T) * 128];                                               \
        __shared__ uint32_t scales[128 * 4 / sizeof(T)];                                                             \
        mx4_quantize_planar<T>(a, codes, scales);                                                                    \
    }                                                                                                                \
    extern "C" __global__ __launch_bounds__(256) void mxq_dequantize_rows_##name(Mx4CodeArgs a) { mx4_dequantize_rows<T>(a); } \
    extern "C" __global__ __launch_bounds__(256) void mxq_dequantize_planar_##name(Mx4CodeArgs a) {                  \
        __shared__ __align__(16) char codes[64 * 4 / sizeof(T) * 128];                                               \
        __shared__ uint32_t scales[128 * 4 / sizeof(T)];                                                             \
        mx4_dequantize_planar<T>(a, codes, scales);                                                                  \
    }                                                                                                                \
    extern "C" __global__ __launch_bounds__(512) void mxq_skinny_##name(Mx4GemmArgs m) { mx4_skinny<T>(m); }         \
    OPS_MX4_D2(name, T, 256, 2, 4)                                                                                   \
    OPS_MX4_D2(name, T, 128, 2, 2)                                                                                   \
    OPS_MX4_D4(name, T, 64, 2, 2)

OPS_MX4_TYPE(bf16, bf16)
OPS_MX4_TYPE(f16, f16)
OPS_MX4_TYPE(f32, float)
