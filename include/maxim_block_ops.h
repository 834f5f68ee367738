/*
 * maxim_block_ops.h - operators of a feed-forward block beside LayerNorm and
 * Dense (maxim_ops.h): the gated Dense, forward and backward.
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
int mxh_gated_workspace(const mxh_mat *x, const mxh_mat *w, const mxh_mat *y, uint64_t *bytes);

/*
 * Its gradients: with dz = (dy * c * act'(a) | dy * act(a)), dx = dz w, dw =
 * dz^T x [2 n][k], db = sum over rows of dz [2 n]. Any of dx, dw and db may be
 * NULL. z has dy's order. As for mxh_dense_backward the products take dz
 * rounded to x's type, db sums it before; db is of x's type or fp32.
 */
int mxh_gated_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w,
                       const mxh_mat *z, int act, float slope, const mxh_mat *dx, const mxh_mat *dw,
                       const mxh_vec *db, void *workspace, uint64_t workspace_bytes);
int mxh_gated_backward_workspace(const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w, const mxh_mat *dx,
                                 const mxh_mat *dw, const mxh_vec *db, uint64_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* MAXIM_BLOCK_OPS_H */
