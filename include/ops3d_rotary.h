/*
 * C ABI of rotary positions along several axes in libops3d_fda.so (gfx950).  No counterpart in the
 * reference.
 *
 * Channel pair p of every head of a token turns by angle = position[axis[p]] * frequency[p]:
 *   (a, b) -> (a cos - b sin, a sin + b cos)
 * HALVES: the pair is channels p and pairs + p; PAIRS: channels 2 p and 2 p + 1.  Channels from 2 pairs
 * on are copied.  With inverse the angle is negated, which is the gradient.
 *
 * Plain pointers and sizes; the launch goes to `stream` (a hipStream_t) and is asynchronous; nothing is
 * allocated.  Return codes as in ops3d_fda.h; dtype F32 / F16 / BF16 is that of x and y.  Angles are formed
 * in 64 bits and reduced there; the product is rounded once.  Base pointers need the alignment of one
 * element only; channels are consecutive, the strides of items, tokens and heads are in elements (an
 * input's may be 0).  y must not overlap x.
 *
 * positions [items or 1, tokens, axes], contiguous, on the device; position_item is the distance between
 * items in elements (0: the same for all).  frequencies and axis_of [pairs] are HOST memory, read before
 * the call returns.  A call has at most OPS3D_ROTARY_MAX_ITEMS items of less than 2^31 tokens, and a token at
 * most 65536 heads, 65536 channels a head and 2^24 channels.
 */
#ifndef OPS3D_ROTARY_H
#define OPS3D_ROTARY_H

#include <stddef.h>
#include <stdint.h>

#include "ops3d_fda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OPS3D_ROTARY_HALVES 0
#define OPS3D_ROTARY_PAIRS 1
#define OPS3D_ROTARY_POSITION_F32 0
#define OPS3D_ROTARY_POSITION_I64 1
#define OPS3D_ROTARY_MAX_PAIRS 128
#define OPS3D_ROTARY_MAX_AXES 8
#define OPS3D_ROTARY_MAX_ITEMS 65535 /* of a call */

/* Writes every channel of y.  strides: {item, token, head}. */
OPS3D_FDA_API int ops3d_rotary(const void *x, const int64_t *x_strides, const void *positions, int position_type,
                               int64_t position_item, const double *frequencies, const int *axis_of, int pairs, int axes,
                               int layout, int inverse, void *y, const int64_t *y_strides, int dtype, int items,
                               int64_t tokens, int heads, int dim, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* OPS3D_ROTARY_H */
