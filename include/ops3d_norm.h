/*
 * C ABI of layer norm over the last axis in libops3d_fda.so (gfx950), and its backward.  No counterpart
 * in the reference, whose callers put torch's norms around the ops.
 *
 *   n[m,c] = (x[m,c] - mean_m) * rstd_m,  rstd_m = 1 / sqrt(var_m + eps)   (var: the mean of squares)
 *   y[m,c] = n[m,c] * weight[c] + bias[c]
 *
 * Plain pointers and sizes; tensors are device memory; launches go to `stream` (a hipStream_t) and are
 * asynchronous; nothing is allocated.  Return codes as in ops3d_fda.h; dtype F32 / F16 / BF16 is that of
 * x, y and their gradients; weight_dtype, which is dtype or F32, that of weight, bias and their
 * gradients.  weight and bias [width] may be NULL (1 and 0).  Statistics and sums are fp32, results are
 * rounded once.  Base pointers need the alignment of one element only.  ld_* are the distances between
 * consecutive rows in elements (0 repeats one row; inputs only); y and grad_x are contiguous.
 *
 * stats: [rows, 3] fp32, written by the forward when not NULL and read by the backward: the mean as the
 * sum of two numbers, and rstd.  Outputs and workspace must overlap neither each other nor an input.
 */
#ifndef OPS3D_NORM_H
#define OPS3D_NORM_H

#include <stddef.h>
#include <stdint.h>

#include "ops3d_fda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Forward: writes every element of y [rows, width]. */
OPS3D_FDA_API int ops3d_layer_norm_forward(const void *x, int64_t ld_x, const void *weight, const void *bias, void *y,
                                           float *stats, int dtype, int weight_dtype, int64_t rows, int width,
                                           float eps, void *stream);

/* Bytes of device workspace (256-byte aligned) the backward needs: partial sums of the weight's and the
 * bias's gradients, of those that are wanted. */
OPS3D_FDA_API size_t ops3d_layer_norm_backward_workspace_bytes(int dtype, int64_t rows, int width, int want_weight,
                                                               int want_bias);

/*
 * Backward, with gw = grad_y * weight:
 *   grad_x[m,c] = rstd_m (gw[m,c] - mean_c(gw) - n[m,c] mean_c(gw n)),
 *   grad_weight[c] = sum_m grad_y[m,c] n[m,c],  grad_bias[c] = sum_m grad_y[m,c]
 * Each written in full; NULL: not wanted.  Results are bitwise repeatable (no atomics).
 */
OPS3D_FDA_API int ops3d_layer_norm_backward(const void *x, int64_t ld_x, const void *weight, const float *stats,
                                            const void *grad_y, int64_t ld_grad_y, void *grad_x, void *grad_weight,
                                            void *grad_bias, void *workspace, size_t workspace_bytes, int dtype,
                                            int weight_dtype, int64_t rows, int width, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* OPS3D_NORM_H */
