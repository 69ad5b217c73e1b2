/*
 * C ABI of the linear operators in libops3d_fda.so (gfx950): a matrix product with bias,
 * activation and residual in its epilogue, for one weight or for weights of their own for groups of
 * consecutive rows, and its backward.  No counterpart in the reference, whose callers use torch's
 * linear layers around the ops (reference tests/test_flash_deform_attn.py:25-60).
 *
 *   z[m,n] = sum_k x[m,k] * weight[g(m)][n,k] + bias[g(m)][n]
 *   y[m,n] = act(z[m,n]) + residual[m,n]
 *
 * Plain pointers and sizes; tensors are device memory; launches go to `stream` (a hipStream_t) and
 * are asynchronous; nothing is allocated.  Return codes as in ops3d_fda.h; dtype F32 / F16 / BF16 is
 * that of every tensor unless stated.  Sums are fp32, rounded once.  Base pointers need the
 * alignment of one element only; rows that start at 16-byte boundaries are faster.
 *
 * Rows: `batch` items of `rows` rows, one after another: row r of item b is row b * rows + r of x,
 * residual, y and the gradients.  ld_* are the distances between consecutive rows in elements
 * (0 repeats one row; read-only tensors only).  weight is [groups, out_features, in_features],
 * contiguous; bias [groups, out_features], contiguous, may be NULL; residual may be NULL.
 *
 * Groups: group_start NULL means one group of all rows (groups must be 1).  Otherwise
 * group_start [group_start_count] int64 on the device, with groups or groups + 1 entries, holds the
 * first row of each group in every item, the same for all items (a level_start_index as it stands);
 * with groups + 1 entries the last is the end of the last group, with groups entries the last group
 * ends with the item.  Groups may be empty.  Entries are read on the device only: each counts as the
 * largest of itself and those before it, held to [0, rows].  Rows in no group (before the first,
 * behind the last) get y = 0 and grad_x = 0, whatever their residual, which has no gradient there
 * (ops3d_linear_keep_rows), and add nothing to the weights' gradients.
 *
 * act_grad: act'(z) for the backward, [batch * rows, out_features], written by the forward when not
 * NULL and read by the backward; fp32 for F32, otherwise a 16-bit code: below 1/8 the bits of the fp16
 * number (11 significant bits), from there on 0x3000 and steps of 2^-14; 0xfe00 is NaN.  Rows in no
 * group are not written.  It must be NULL for OPS3D_LINEAR_ACT_NONE.
 *
 * Outputs and workspace must overlap neither each other nor an input (a residual neither): some results
 * are computed by two blocks, which write the same value.
 */
#ifndef OPS3D_LINEAR_H
#define OPS3D_LINEAR_H

#include <stddef.h>
#include <stdint.h>

#include "ops3d_fda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OPS3D_LINEAR_ACT_NONE 0
#define OPS3D_LINEAR_ACT_RELU 1
#define OPS3D_LINEAR_ACT_GELU 2      /* 0.5 z (1 + erf(z / sqrt 2)) */
#define OPS3D_LINEAR_ACT_GELU_TANH 3 /* 0.5 z (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) */
#define OPS3D_LINEAR_ACT_SILU 4      /* z / (1 + exp(-z)) */
#define OPS3D_LINEAR_MAX_GROUPS 4096

/* Bytes of device workspace (256-byte aligned) the forward needs: parts of long sums over few tiles; 0
 * for other sizes and for invalid ones. */
OPS3D_FDA_API size_t ops3d_linear_forward_workspace_bytes(int dtype, int batch, int64_t rows, int groups,
                                                          int out_features, int in_features, int grouped);

/* Forward: writes every element of y ([batch * rows, out_features], contiguous). */
OPS3D_FDA_API int ops3d_linear_forward(const void *x, int64_t ld_x, const void *weight, const void *bias,
                                       const void *residual, int64_t ld_residual, const int64_t *group_start,
                                       int group_start_count, void *y, void *act_grad, void *workspace,
                                       size_t workspace_bytes, int dtype, int act, int batch, int64_t rows, int groups,
                                       int out_features, int in_features, void *stream);

#define OPS3D_LINEAR_WANT_X 1
#define OPS3D_LINEAR_WANT_WEIGHT 2
#define OPS3D_LINEAR_WANT_BIAS 4

/* Bytes of device workspace (256-byte aligned) the backward needs for the gradients in `want` (the
 * outputs that are not NULL): dz (with an act_grad, for grad_weight and grad_bias) and partial sums, of
 * grad_x over parts of long sums and of the other two over chunks of rows. */
OPS3D_FDA_API size_t ops3d_linear_backward_workspace_bytes_for(int dtype, int batch, int64_t rows, int groups,
                                                               int out_features, int in_features, int grouped,
                                                               int with_act_grad, int want);

/* The same for all three. */
OPS3D_FDA_API size_t ops3d_linear_backward_workspace_bytes(int dtype, int batch, int64_t rows, int groups,
                                                           int out_features, int in_features, int grouped,
                                                           int with_act_grad);

/*
 * Backward.  With dz = grad_y * act_grad (grad_y where act_grad is NULL):
 *   grad_x[m,k] = sum_n dz[m,n] weight[g(m)][n,k]   [batch * rows, in_features]
 *   grad_weight[g][n,k] = sum_{m in g} dz[m,n] x[m,k],  grad_bias[g][n] = sum_{m in g} dz[m,n]
 * Each written in full, contiguous; NULL: not wanted.  weight is read for grad_x only and x for
 * grad_weight and grad_bias only.  dz is rounded to dtype before it is multiplied or summed.  Results
 * are bitwise repeatable (no atomics).
 */
OPS3D_FDA_API int ops3d_linear_backward(const void *x, int64_t ld_x, const void *weight, const int64_t *group_start,
                                        int group_start_count, const void *act_grad, const void *grad_y,
                                        int64_t ld_grad_y, void *grad_x, void *grad_weight, void *grad_bias,
                                        void *workspace, size_t workspace_bytes, int dtype, int batch, int64_t rows,
                                        int groups, int out_features, int in_features, void *stream);

/*
 * dst = src in rows of a group, 0 in rows of none ([batch * rows, features], contiguous): the gradient of
 * a residual, which is grad_y in the former only, since y is 0 in the latter.  Without groups it is grad_y.
 */
OPS3D_FDA_API int ops3d_linear_keep_rows(const void *src, int64_t ld_src, const int64_t *group_start,
                                         int group_start_count, void *dst, int dtype, int batch, int64_t rows,
                                         int groups, int features, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* OPS3D_LINEAR_H */
