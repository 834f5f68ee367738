/*
 * maxim_ops.h - LayerNorm and Dense on a caller's own device tensors, forward
 * and backward, as hand-written gfx950 kernels.
 *
 * The executor (maxim_hip.h) runs one inference plan over its own fp32 arena.
 * These calls are for the programs beside it: training and serving token models,
 * or tuning the LayerNorm and Dense layers of a MAXIM checkpoint's blocks (the
 * gradients of its convolutions, gates and resizing are the program's own), in
 * fp32, fp16 or bf16. No counterpart in the reference, which has no gradients
 * and no 16-bit types.
 *
 * Matrices are views: rows are positions (pixels or tokens), columns features,
 * `row_stride` and `col_stride` elements apart, one of the two 1. So the
 * executor's planar [c][h][w] order is (row_stride 1, col_stride h * w) and a
 * token-major [n][c] array (row_stride c, col_stride 1); slices of wider
 * buffers and broadcast inputs (a stride of 0) need no copy. Any alignment of
 * the element, any sizes whose launches have fewer than 2^32 threads each (a
 * call with a larger one is refused: some of 2^24 features or 2^27 positions and
 * more). An output's own elements must not share storage, and an output must
 * not overlap any other operand, but where a call says so.
 *
 * Sums, means and variances are fp32; a result is rounded once, to nearest
 * even, when it is stored. fp32 products are formed on the bf16 matrix cores
 * from three bf16 parts of each operand (every bit of a float, whatever its
 * size; one product is off by 1.82e-7 of itself at most), and sums that are not
 * finite again in fp32, so infinities and NaN are fp32's. No atomics: the same
 * call gives the same bits.
 *
 * Every call is asynchronous, in stream order on `stream` (a hipStream_t of
 * `device`; NULL: the device's default stream). It allocates nothing and
 * records only kernel nodes, so a capture of the stream holds it. Before a
 * capture, mxh_ops_ready(device) has to have loaded the kernels once. The
 * calling thread's current device is left as it was.
 *
 * Where a call needs scratch, `workspace` is device memory of at least the
 * bytes that its _workspace function gives for the same operands, 16-byte
 * aligned and apart from all of them; the call owns it until the stream has
 * passed. Two calls may share
 * it in stream order; calls (or captured graphs) that can overlap need one
 * each.
 *
 * Errors: negative status, message in mx_last_error(); a refused call has
 * launched nothing.
 */
#ifndef MAXIM_OPS_H
#define MAXIM_OPS_H

#include <stdint.h>

#include "maxim_plan.h"

#ifdef __cplusplus
extern "C" {
#endif

enum mxh_dtype { MXH_F32 = 0, MXH_F16 = 1, MXH_BF16 = 2 };

/* gelu is x Phi(x) (the executor's), gelu_tanh its tanh form, silu
 * x / (1 + e^-x), lrelu x or slope * x for x < 0 (slope 0: ReLU). */
enum mxh_act { MXH_NONE = 0, MXH_GELU = 1, MXH_GELU_TANH = 2, MXH_SILU = 3, MXH_LRELU = 4, MXH_SIGMOID = 5 };

typedef struct mxh_mat {
    void *data;
    int64_t rows, cols, row_stride, col_stride;
    int32_t dtype, reserved;
} mxh_mat;

/* A contiguous vector: a parameter or its gradient. */
typedef struct mxh_vec {
    void *data;
    int64_t n;
    int32_t dtype, reserved;
} mxh_vec;

/* Load the kernels on `device` (done by the first call otherwise). */
int mxh_ops_ready(int device);

/*
 * y = (x - mean) * rstd * scale + bias over each row's columns, rstd =
 * 1 / sqrt(variance + eps), the variance taken about the mean. bias may be
 * NULL. mean and rstd ([rows] fp32 each, NULL: not kept) are what the
 * backward pass takes. y has x's type and memory order and may be x itself.
 * scale and bias are both of x's type or both fp32.
 */
int mxh_layernorm(int device, void *stream, const mxh_mat *x, const mxh_vec *scale, const mxh_vec *bias, float eps,
                  const mxh_mat *y, float *mean, float *rstd);

/*
 * With xh = (x - mean) * rstd and g = dy * scale:
 *   dx = rstd * (g - mean(g) - xh * mean(g * xh)) + add   (means over a row)
 *   dscale = sum over rows of dy * xh, dbias = sum over rows of dy
 * add (the gradient that reaches x past the LayerNorm, as a residual
 * connection's) may be NULL; so may dx, or dscale and dbias (both or
 * neither). dx may be dy or add itself. dscale and dbias have scale's type.
 * All matrices have x's type and order.
 */
int mxh_layernorm_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_vec *scale,
                           const float *mean, const float *rstd, const mxh_mat *add, const mxh_mat *dx,
                           const mxh_vec *dscale, const mxh_vec *dbias, void *workspace, uint64_t workspace_bytes);
int mxh_layernorm_backward_workspace(const mxh_mat *x, uint64_t *bytes);

/*
 * z = x w^T + bias, y = act(z) + residual: x [rows][k], w [n][k] (a
 * checkpoint's Dense kernel [k][n] is the same view with its strides
 * exchanged), y [rows][n]. bias (of x's type or fp32), residual and z (kept
 * for the backward pass) may be NULL. All matrices have x's type; residual
 * and z have y's order, x and w any. y may be the residual itself.
 */
int mxh_dense(int device, void *stream, const mxh_mat *x, const mxh_mat *w, const mxh_vec *bias, int act, float slope,
              const mxh_mat *residual, const mxh_mat *y, const mxh_mat *z, void *workspace, uint64_t workspace_bytes);
int mxh_dense_workspace(const mxh_mat *x, const mxh_mat *w, const mxh_mat *y, uint64_t *bytes);

/*
 * The gradients of y = act(x w^T + bias) + residual from dy: with
 * dz = dy * act'(z), dx = dz w, dw = dz^T x, db = sum over rows of dz (the
 * residual's gradient is dy itself). Any of dx, dw and db may be NULL. z is
 * the forward pass's, of dy's order; NULL when act is MXH_NONE. The products
 * take dz rounded to x's type (in fp16 a dz past 65504 is infinite), db sums it
 * before the rounding. db is of x's type or fp32.
 */
int mxh_dense_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w,
                       const mxh_mat *z, int act, float slope, const mxh_mat *dx, const mxh_mat *dw,
                       const mxh_vec *db, void *workspace, uint64_t workspace_bytes);
int mxh_dense_backward_workspace(const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w, int act, const mxh_mat *dx,
                                 const mxh_mat *dw, const mxh_vec *db, uint64_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* MAXIM_OPS_H */
