// Rotary positions along several axes (gfx950; include/ops3d_rotary.h).
//
// The bytes bound it: x in, y out.  A block has some tokens: it forms their angles' cosines and sines in
// LDS first, one pair of a token a thread at a time, since every head of a token turns by the same ones, then
// streams the heads in 16-byte chunks.  The angle in turns is a 64-bit product, and its whole turns are dropped
// there: positions far out lose nothing.
//
// 73728 tokens, 16 heads of 32, three axes, bf16: 31.6 us (151 MB at 4.8 TB/s; a copy of 256 MB reaches 5.4); 2 x 1551
// tokens, 20 heads of 128, pairs, fp16: 10.3 (31.8 MB, 3.1).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/ops3d_rotary.h"
#include "elements.h"

namespace ops3d_fda {
int set_last_error(int code, const char *text);   // fda_capi.hip
}

namespace {

using namespace ops3d_elements;

struct Args {
  const void *x;
  void *y;
  const void *positions;
  int64_t x_item, x_token, x_head, y_item, y_token, y_head, pos_item;
  int64_t tokens;
  int heads, dim, pairs, axes, per_block;
  float sign;
  double turns[OPS3D_ROTARY_MAX_PAIRS];   // frequency / 2 pi
  uint8_t axis[OPS3D_ROTARY_MAX_PAIRS];
};

constexpr int kTable = 2048;   // pairs of a block's tokens

// VEC: whole chunks of 16 bytes; otherwise single pairs and channels.
template <typename T, typename P, bool PAIRS, bool VEC> __global__ __launch_bounds__(256) void rotary_kernel(Args p) {
  constexpr int CH = 16 / (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) float cs[kTable], sn[kTable];
  const int64_t t0 = (int64_t)blockIdx.x * p.per_block;
  const int item = blockIdx.y, nt = (int)min((int64_t)p.per_block, p.tokens - t0);
  const P *pos = static_cast<const P *>(p.positions) + item * p.pos_item + t0 * p.axes;
  for (int i = threadIdx.x; i < nt * p.pairs; i += 256) {
    const int t = i / p.pairs, k = i - t * p.pairs;
    const double turn = (double)pos[t * p.axes + p.axis[k]] * p.turns[k];
    const float half = (float)(2.0 * (turn - rint(turn)));   // half turns, in [-1, 1]
    float s, c;
    sincospif(half, &s, &c);
    cs[i] = c;
    sn[i] = s * p.sign;
  }
  __syncthreads();
  const T *x = static_cast<const T *>(p.x) + item * p.x_item + t0 * p.x_token;
  T *y = static_cast<T *>(p.y) + item * p.y_item + t0 * p.y_token;
  // a head's units: those of its pairs, then those of the channels that are copied
  constexpr int kUnit = VEC ? (PAIRS ? CH / 2 : CH) : 1, kCopy = VEC ? CH : 1;
  const int turned = p.pairs / kUnit, units = turned + (p.dim - 2 * p.pairs) / kCopy;
  const int all = nt * p.heads * units;
  for (int i = threadIdx.x; i < all; i += 256) {
    const int th = i / units, u = i - th * units, t = th / p.heads, h = th - t * p.heads;
    const T *from = x + t * p.x_token + h * p.x_head;
    T *to = y + t * p.y_token + h * p.y_head;
    if (u >= turned) {
      const int c = 2 * p.pairs + (u - turned) * kCopy;
      if constexpr (VEC) store16(to + c, load16(from + c));
      else to[c] = from[c];
      continue;
    }
    const float *cu = cs + t * p.pairs + u * kUnit, *su = sn + t * p.pairs + u * kUnit;
    if constexpr (!VEC) {
      const int ia = PAIRS ? 2 * u : u, ib = PAIRS ? 2 * u + 1 : p.pairs + u;
      const float a = (float)from[ia], b = (float)from[ib];
      to[ia] = (T)(a * *cu - b * *su);
      to[ib] = (T)(a * *su + b * *cu);
    } else if constexpr (PAIRS) {
      Chunk<T> c;
      c.raw = load16(from + u * CH);
#pragma unroll
      for (int k = 0; k < CH / 2; ++k) {
        const float a = (float)c.e[2 * k], b = (float)c.e[2 * k + 1];
        c.e[2 * k] = (T)(a * cu[k] - b * su[k]);
        c.e[2 * k + 1] = (T)(a * su[k] + b * cu[k]);
      }
      store16(to + u * CH, c.raw);
    } else {
      Chunk<T> ca, cb;
      ca.raw = load16(from + u * CH);
      cb.raw = load16(from + p.pairs + u * CH);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const float a = (float)ca.e[k], b = (float)cb.e[k];
        ca.e[k] = (T)(a * cu[k] - b * su[k]);
        cb.e[k] = (T)(a * su[k] + b * cu[k]);
      }
      store16(to + u * CH, ca.raw);
      store16(to + p.pairs + u * CH, cb.raw);
    }
  }
}

int fail(int code, const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return ops3d_fda::set_last_error(code, buf);
}
int elem_size(int dtype) {
  return dtype == OPS3D_FDA_F32 ? 4 : dtype == OPS3D_FDA_F16 || dtype == OPS3D_FDA_BF16 ? 2 : 0;
}

template <typename T, typename P> hipError_t launch(const Args &a, int layout, dim3 grid, hipStream_t st) {
  constexpr int CH = 16 / (int)sizeof(T);
  const bool vec = a.dim % CH == 0 && a.pairs % (layout == OPS3D_ROTARY_PAIRS ? CH / 2 : CH) == 0;
  if (layout == OPS3D_ROTARY_PAIRS) {
    if (vec) rotary_kernel<T, P, true, true><<<grid, 256, 0, st>>>(a);
    else rotary_kernel<T, P, true, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (vec) rotary_kernel<T, P, false, true><<<grid, 256, 0, st>>>(a);
    else rotary_kernel<T, P, false, false><<<grid, 256, 0, st>>>(a);
  }
  return hipGetLastError();
}
template <typename T> hipError_t launch_type(const Args &a, int layout, int position_type, dim3 grid, hipStream_t st) {
  return position_type == OPS3D_ROTARY_POSITION_F32 ? launch<T, float>(a, layout, grid, st)
                                                    : launch<T, int64_t>(a, layout, grid, st);
}

}  // namespace

extern "C" int ops3d_rotary(const void *x, const int64_t *x_strides, const void *positions, int position_type,
                            int64_t position_item, const double *frequencies, const int *axis_of, int pairs, int axes,
                            int layout, int inverse, void *y, const int64_t *y_strides, int dtype, int items,
                            int64_t tokens, int heads, int dim, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  const int es = elem_size(dtype);
  if (!es) return fail(OPS3D_FDA_EINVAL, "unsupported dtype code %d", dtype);
  if (position_type != OPS3D_ROTARY_POSITION_F32 && position_type != OPS3D_ROTARY_POSITION_I64)
    return fail(OPS3D_FDA_EINVAL, "unknown position type %d", position_type);
  if (layout != OPS3D_ROTARY_HALVES && layout != OPS3D_ROTARY_PAIRS) return fail(OPS3D_FDA_EINVAL, "unknown layout %d", layout);
  if (items < 0 || tokens < 0 || heads < 0 || items > OPS3D_ROTARY_MAX_ITEMS || tokens > 0x7fffffff || heads > 65536)
    return fail(OPS3D_FDA_EINVAL, "invalid or too many items, tokens or heads: %d, %lld, %d", items, (long long)tokens, heads);
  if (dim < 1 || dim > 65536) return fail(OPS3D_FDA_EINVAL, "heads must have 1..65536 channels, got %d", dim);
  if ((int64_t)heads * dim > 1 << 24)
    return fail(OPS3D_FDA_EINVAL, "a token has at most 2^24 channels, got %d heads of %d", heads, dim);
  if (axes < 1 || axes > OPS3D_ROTARY_MAX_AXES)
    return fail(OPS3D_FDA_EINVAL, "positions must have 1..%d axes, got %d", OPS3D_ROTARY_MAX_AXES, axes);
  if (pairs < 0 || pairs > OPS3D_ROTARY_MAX_PAIRS || 2 * pairs > dim)
    return fail(OPS3D_FDA_EINVAL, "%d pairs do not fit heads of %d channels, or are more than %d", pairs, dim, OPS3D_ROTARY_MAX_PAIRS);
  if (!x_strides || !y_strides || (pairs && (!frequencies || !axis_of))) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  for (int i = 0; i < pairs; ++i) {
    if (axis_of[i] < 0 || axis_of[i] >= axes) return fail(OPS3D_FDA_EINVAL, "pair %d has axis %d of %d", i, axis_of[i], axes);
    if (!isfinite(frequencies[i])) return fail(OPS3D_FDA_EINVAL, "the frequency of pair %d is not finite", i);
  }
  if (items == 0 || tokens == 0 || heads == 0) return OPS3D_FDA_OK;
  if (!x || !y || !positions) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  const auto off = [](const void *q, int n) { return (reinterpret_cast<uintptr_t>(q) & (uintptr_t)(n - 1)) != 0; };
  if (off(x, es) || off(y, es) || off(positions, position_type == OPS3D_ROTARY_POSITION_F32 ? 4 : 8))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  Args a{};
  a.x = x;
  a.y = y;
  a.positions = positions;
  a.x_item = x_strides[0], a.x_token = x_strides[1], a.x_head = x_strides[2];
  a.y_item = y_strides[0], a.y_token = y_strides[1], a.y_head = y_strides[2];
  a.pos_item = position_item;
  a.tokens = tokens;
  a.heads = heads;
  a.dim = dim;
  a.pairs = pairs;
  a.axes = axes;
  a.sign = inverse ? -1.f : 1.f;
  for (int i = 0; i < pairs; ++i) {
    a.turns[i] = frequencies[i] * 0.15915494309189533577;
    a.axis[i] = (uint8_t)axis_of[i];
  }
  // tokens a block: about 16 KB of channels, within the table
  int64_t n = 16384 / ((int64_t)heads * dim * es);
  if (pairs && n > kTable / pairs) n = kTable / pairs;
  a.per_block = (int)(n < 1 ? 1 : n > 256 ? 256 : n);
  const dim3 grid((unsigned)((tokens + a.per_block - 1) / a.per_block), (unsigned)items);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = dtype == OPS3D_FDA_F32   ? launch_type<float>(a, layout, position_type, grid, st)
                       : dtype == OPS3D_FDA_F16 ? launch_type<_Float16>(a, layout, position_type, grid, st)
                                                : launch_type<__bf16>(a, layout, position_type, grid, st);
  if (e == hipSuccess) return OPS3D_FDA_OK;
  return fail(OPS3D_FDA_ERUNTIME, "rotary positions: kernel launch failed: %s", hipGetErrorString(e));
}
