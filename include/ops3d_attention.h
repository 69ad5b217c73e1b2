/*
 * C ABI of attention over all tokens in libops3d_fda.so (gfx950), with grouped heads, causal or not, over
 * items of a batch or over sequences packed one behind another, and its backward.  No counterpart in the
 * reference, whose attention samples a few places of the value.
 *
 *   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j) / sum_j' exp(scale q_i.k_j')
 *
 * over the keys j that query i of the same sequence sees: all, or, causal, those with
 * j <= i + (keys - queries), so that the last query sees all.  A query that sees none gets 0.  Query head h
 * reads key and value head h / (heads / kv_heads).
 *
 * Plain pointers and sizes; tensors are device memory; launches go to `stream` (a hipStream_t) and are
 * asynchronous; nothing is allocated.  Return codes as in ops3d_fda.h; dtype F32 / F16 / BF16 is that of
 * every tensor.  Logits, their statistics and all sums are fp32; probabilities and the gradients of logits
 * are rounded to dtype before they are multiplied; results are rounded once.  Base pointers need the
 * alignment of one element only; channels are consecutive, and rows that start at 16-byte boundaries are
 * faster.
 *
 * Two forms.  Items (q_start NULL): `items` items of q_rows queries and k_rows keys each, of which q_len
 * and k_len [items] int64 on the device, where not NULL, say how many count (held to [0, rows]).  Packed
 * (q_start not NULL): items must be 1; q_start and k_start hold the first rows of `sequences` sequences,
 * with sequences or sequences + 1 entries each; with sequences entries the last one ends with the rows.
 * Entries are read on the device only: each counts as the largest of itself and those before it, held to
 * [0, rows].  Sequences may be empty.  Rows that do not count or are in no sequence are not read; their
 * outputs and gradients are 0.  Outputs and workspace must overlap neither each other nor an input.
 *
 * A query whose visible logits are all minus infinity, or of which one is NaN, gives NaN.  In fp16 probabilities and
 * the gradients of logits are held times powers of two, the latter's chosen for each query and each key, so that they keep
 * their precision where they are small and do not overflow where they are large.
 *
 * Limits: OPS3D_ATTENTION_MAX_DIM channels, OPS3D_ATTENTION_MAX_SEQUENCES packed sequences or 2^24 items, less than
 * 2^31 - 65536 keys, and queries times the heads of a group, of an item.
 */
#ifndef OPS3D_ATTENTION_H
#define OPS3D_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#include "ops3d_fda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OPS3D_ATTENTION_MAX_DIM 128
#define OPS3D_ATTENTION_MAX_SEQUENCES 65536

/* A tensor [item, token, head, channel]; strides in elements (an input's may be 0). */
typedef struct ops3d_attention_tensor {
  void *data;
  int64_t item, token, head;
} ops3d_attention_tensor;

typedef struct ops3d_attention_problem {
  const int64_t *q_start, *k_start, *q_len, *k_len;
  int64_t q_rows, k_rows;
  int32_t q_start_count, k_start_count;
  int32_t sequences, items;
  int32_t heads, kv_heads, dim;
  int32_t dtype, causal;
  float scale; /* positive */
} ops3d_attention_problem;

/* Bytes of device workspace (256-byte aligned) of the forward, to be asked for each problem: partial results where
 * the keys are cut into parts (few queries that see many keys; causal or packed problems of middling size), and the
 * table of tiles of more than 64 packed sequences.  0 where neither is needed, and for invalid sizes. */
OPS3D_FDA_API size_t ops3d_attention_forward_workspace_bytes(const ops3d_attention_problem *problem);

/* Writes every channel of out.  For the backward, where not NULL: lse [items, heads, q_rows] fp32 (in an order of
 * the library's own), and out_rest [items, q_rows, heads, dim], contiguous, of dtype: what rounding took from
 * out. */
OPS3D_FDA_API int ops3d_attention_forward(const ops3d_attention_problem *problem, const ops3d_attention_tensor *q,
                                          const ops3d_attention_tensor *k, const ops3d_attention_tensor *v,
                                          const ops3d_attention_tensor *out, void *out_rest, float *lse, void *workspace,
                                          size_t workspace_bytes, void *stream);

/* Bytes of device workspace (256-byte aligned) of the backward: the products of out with grad_out, partial sums
 * where a side is cut into parts, and the table of tiles of more than 64 packed sequences. */
OPS3D_FDA_API size_t ops3d_attention_backward_workspace_bytes(const ops3d_attention_problem *problem);

/* Writes every channel of grad_q, grad_k and grad_v; grad_q may be NULL, and grad_k and grad_v together:
 * not wanted.  out_rest may be NULL; with it, the products of out with grad_out are those of the unrounded
 * output, and the gradients of logits are closer.  Results are bitwise repeatable (no atomics). */
OPS3D_FDA_API int ops3d_attention_backward(const ops3d_attention_problem *problem, const ops3d_attention_tensor *q,
                                           const ops3d_attention_tensor *k, const ops3d_attention_tensor *v,
                                           const ops3d_attention_tensor *out, const void *out_rest, const float *lse,
                                           const ops3d_attention_tensor *grad_out, const ops3d_attention_tensor *grad_q,
                                           const ops3d_attention_tensor *grad_k, const ops3d_attention_tensor *grad_v,
                                           void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* OPS3D_ATTENTION_H */
