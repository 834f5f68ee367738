/*
 * maxim_block_ops.h - operators of a feed-forward block beside LayerNorm and
 * Dense (maxim_ops.h): the gated Dense, forward and backward; the gradients'
 * global norm and clipping, between a backward pass and the optimizer; and
 * Dense with weights in 4-bit blocks, for serving.
 *
 * Everything that maxim_ops.h says of operands, alignment, sizes, precision,
 * streams, captures, workspaces and errors holds here too; mxh_ops_ready loads
 * these kernels as well. No counterpart in the reference.
 */
#ifndef MAXIM_BLOCK_OPS_H
#define MAXIM_BLOCK_OPS_H

#include "maxim_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The gated Dense of a feed-forward block: z = x w^T + bias with the gate's n
 * features first and then the values', z = (a | c), and y = act(a) * c. x
 * [rows][k], w [2 n][k], bias [2 n], y [rows][n], z [rows][2 n] (NULL: not
 * kept; the backward pass takes it). One launch where the sums are not cut:
 * without z nothing but y is written. x, y and z have one type and memory
 * order; w may lie either way.
 */
int mxh_gated(int device, void *stream, const mxh_mat *x, const mxh_mat *w, const mxh_vec *bias, int act, float slope,
              const mxh_mat *y, const mxh_mat *z, void *workspace, uint64_t workspace_bytes);
int mxh_gated_workspace(const mxh_mat *x, const mxh_mat *w, const mxh_mat *y, const mxh_mat *z, uint64_t *bytes);

/*
 * Its gradients: with dz = (dy * c * act'(a) | dy * act(a)), dx = dz w, dw =
 * dz^T x [2 n][k], db = sum over rows of dz [2 n]. Any of dx, dw and db may be
 * NULL. z has dy's order. As for mxh_dense_backward the products take dz
 * rounded to x's type, db sums it before; db is of x's type or fp32. In bf16
 * that is one rounding more, half a step of each term, than dz in fp32 would
 * have: dx and dw of 4096 x 1024 to 2 x 2048 are 2.35e-3 off in the mean, not
 * 1.66e-3; operands cast to fp32 are without it. In fp16 dz keeps to the type's
 * range where its terms would not: with the largest finite one below 1 or past
 * 65504 all are taken times one power of two, and the sums divided by it. Each
 * is off by half a step of its own, or by 2^-25 as it is and by 2^-39 of the
 * largest (2^-85 at least) where it was scaled.
 */
int mxh_gated_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w,
                       const mxh_mat *z, int act, float slope, const mxh_mat *dx, const mxh_mat *dw,
                       const mxh_vec *db, void *workspace, uint64_t workspace_bytes);
int mxh_gated_backward_workspace(const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w, const mxh_mat *dx,
                                 const mxh_mat *dw, const mxh_vec *db, uint64_t *bytes);

/*
 * The global norm of a list of gradients, N = sqrt(sum of all elements'
 * squares), as one fp32 value on the device (0 of no elements). `grads` is
 * host memory: `count` contiguous tensors of any types and sizes, zero among
 * them; the call has read it when it returns. Squares and their sums are
 * formed in 64 bits, so N is rounded once and infinite only past fp32's range,
 * or with an infinity among the elements (NaN with a NaN).
 */
int mxh_grad_norm(int device, void *stream, const mxh_vec *grads, int64_t count, float *norm, void *workspace,
                  uint64_t workspace_bytes);
int mxh_grad_norm_workspace(const mxh_vec *grads, int64_t count, uint64_t *bytes);

/*
 * The same, and out[i] = grads[i] * (max_norm / N) where N > max_norm; else,
 * and where N is not finite (a step that the caller skips), out[i] = grads[i].
 * out NULL, or an out[i].data of grads[i].data: in place, with nothing written
 * where nothing changes. Each out[i] has its gradient's size and type and lies
 * apart from every other tensor. mxh_grad_norm_workspace gives the bytes.
 */
int mxh_grad_clip(int device, void *stream, const mxh_vec *grads, const mxh_vec *out, int64_t count, float max_norm,
                  float *norm, void *workspace, uint64_t workspace_bytes);
/* By a norm on the device that the caller has, as one added up over ranks. */
int mxh_grad_clip_by(int device, void *stream, const mxh_vec *grads, const mxh_vec *out, int64_t count, float max_norm,
                     const float *norm);

/*
 * A matrix [rows][cols] in blocks of 32 features with 4 bits an element (1
 * sign, 2 exponent, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and a scale of
 * 8 bits, 2^(s - 127), 255 for NaN: 17 bytes for 32 elements.
 *
 * codes: a line of ceil(cols / 256) * 128 bytes a row, an element's code in the
 * low half of its byte where its feature is even; scales: for 64 rows and 256
 * features 512 bytes, that of row r and block b at [r / 64][b / 8][b % 4][r %
 * 16][r / 16 % 4][b / 4 % 2]. Elements past the last feature and scales past
 * the last row are 0. Both are 16-byte aligned; mxh_mx4_size gives their bytes.
 */
typedef struct mxh_mx4 {
    void *codes, *scales;
    int64_t rows, cols;
} mxh_mx4;
int mxh_mx4_size(int64_t rows, int64_t cols, uint64_t *codes, uint64_t *scales);

/*
 * With m a block's largest magnitude: s - 127 = floor(log2 m) - 2, at least
 * -127, and each element is x / 2^(s - 127) rounded to the nearest code, ties to
 * even, 6 at most. A block with an infinity or a NaN is NaN. x of any type and
 * either memory order; back, each value is rounded to y's type.
 */
int mxh_mx4_quantize(int device, void *stream, const mxh_mat *x, const mxh_mx4 *q);
int mxh_mx4_dequantize(int device, void *stream, const mxh_mx4 *q, const mxh_mat *y);

/*
 * y = act(X W^T + bias) + residual with W = w [n][k] and X = x [rows][k] in the
 * values of 4-bit blocks, x quantised in the call, the products on the matrix
 * cores and summed in fp32. bias (of x's type or fp32) and residual may be
 * NULL. residual and y have x's type and one memory order, x any. y may be the
 * residual itself.
 */
int mxh_mx4_dense(int device, void *stream, const mxh_mat *x, const mxh_mx4 *w, const mxh_vec *bias, int act, float slope,
                  const mxh_mat *residual, const mxh_mat *y, void *workspace, uint64_t workspace_bytes);
int mxh_mx4_dense_workspace(const mxh_mat *x, const mxh_mx4 *w, const mxh_mat *residual, const mxh_mat *y,
                            uint64_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* MAXIM_BLOCK_OPS_H */
