// Argument blocks of the training and serving operators' kernels, shared by
// the host side (g++) and the gfx950 kernels (hipcc): 8-byte fields first,
// then 4-byte fields in pairs, each kernel taking one block by value.
#pragma once

#include <stdint.h>

// Element types, include/maxim_ops.h's mxh_dtype.
enum { MXO_F32 = 0, MXO_F16 = 1, MXO_BF16 = 2 };

// Activations, include/maxim_ops.h's mxh_act.
enum { MXO_NONE = 0, MXO_GELU, MXO_GELU_TANH, MXO_SILU, MXO_LRELU, MXO_SIGMOID };

// C[m][n] = act(sum_k A(m, k) B(n, k) + bias) + residual, n contiguous in C,
// in the residual and in z (the sum with its bias, when kept). Each of A and
// B is contiguous along k or along its other axis (the kernel's form), `ld`
// elements apart along the other one.
struct OpsGemmArgs {
    const void *a, *b, *bias, *res;
    void *c, *z;
    float *part;  // [splits][m][n] partial sums when splits > 1
    const float *back;  // fp16: sums are times *back (null: as they are)
    int64_t lda, ldb, ldc, ldr, ldz;
    int32_t m, n, k;
    int32_t splits, kchunk;  // split s covers k in [s kchunk, (s + 1) kchunk)
    int32_t tiles_m, tiles_n;
    int32_t act;
    float slope;
    int32_t bias_f32;   // the bias is fp32, else of the operands' type
    int32_t bias_rows, pad;  // one bias value per m instead of per n
};

// Operands of a product copied to lines of whole 16 bytes, zeros at their
// ends: job blockIdx.y, 2^shift threads a line, four vectors each, `segs` such
// runs a line.
struct OpsPackJob {
    const void *src;
    void *dst;
    int64_t lines, extent, src_ld, dst_ld;
    int32_t shift, segs;
};
struct OpsPackArgs {
    OpsPackJob job[2];
};

// x, y and the gradients [rows][cols] at rs and cs elements between rows and
// columns, one of them 1.
struct OpsLnArgs {
    const void *x, *scale, *bias;
    void *y;
    float *mean, *rstd;
    int64_t rows, cols;
    int64_t xrs, xcs, yrs, ycs;
    float eps;
    int32_t param_f32;
};

struct OpsLnBwdArgs {
    const void *dy, *x, *scale, *add;
    const float *mean, *rstd;
    void *dx;
    float *part;  // [nparts][2][cols]: dscale's and dbias's partial sums
    int64_t rows, cols;
    int64_t dyrs, dycs, xrs, xcs, ars, acs, dxrs, dxcs;
    int32_t nparts, param_f32;
};

// dz = dy act'(z), and the partial sums of dz over the rows.
struct OpsDzArgs {
    const void *dy, *z;
    void *dz;     // null: only the sums
    float *part;  // [nparts][cols]; null: no sums
    int64_t rows, cols;
    int64_t dyrs, dycs, zrs, zcs, drs, dcs;
    int32_t nparts, act;
    float slope;
    int32_t pad;
};

// out[i] = sum over p of part[p][i] (a second result's parts follow each
// first's: [nparts][nout][n]).
struct OpsJoinArgs {
    const float *part;
    void *out0, *out1;
    int64_t n;
    int32_t nparts, nout;
    int32_t dtype, pad;
};

// A gradient's two joins in one launch: a product's splits (`g`, to g.c; blocks
// from 0) and the bias's partial sums (blocks from `first`).
struct OpsGradJoinArgs {
    OpsGemmArgs g;
    const float *part;
    void *out;
    int32_t n, nparts;
    int32_t first, dtype;
};

// The gated Dense's dz pass: z and dz have twice dy's features, cols the half's.
// A single part needs no joining: its sums are the bias's gradient. fp16: each
// block's largest finite |dz| goes to `top`, where the launch that follows finds
// the scale that dz needs.
enum { MXO_DZ = 0, MXO_DZ_SCALED, MXO_DZ_TOPS };
struct OpsGatedDzArgs {
    OpsDzArgs d;
    void *db;     // null: the sums go to d.part
    float *top;   // [ntop], and one more for all of them; null: none are kept
    float *back;  // what the products take dz's scale back by
    int32_t db_type, pass;
    int32_t ntop, pad;
};
