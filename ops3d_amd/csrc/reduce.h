// Sums and maxima over the lanes of a wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ops3d_reduce {

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
struct Add {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Max {
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// v of the lane 16 or 32 lanes away, combined with this lane's.
template <typename OP> __device__ __forceinline__ float across16(float v) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return OP::of(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
template <typename OP> __device__ __forceinline__ float across32(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return OP::of(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// Over aligned groups of L lanes, the same bits in every lane of one: neighbours, neighbouring pairs,
// then the mirror images of 8 and 16 lanes, whose halves are uniform by then.  All of a group's lanes
// are active.
template <int L, typename OP> __device__ __forceinline__ float all(float v) {
  if (L >= 2) v = OP::of(v, dpp<0xb1>(v));
  if (L >= 4) v = OP::of(v, dpp<0x4e>(v));
  if (L >= 8) v = OP::of(v, dpp<0x141>(v));
  if (L >= 16) v = OP::of(v, dpp<0x140>(v));
  if (L >= 32) v = across16<OP>(v);
  if (L >= 64) v = across32<OP>(v);
  return v;
}
template <int L> __device__ __forceinline__ float sum(float v) { return all<L, Add>(v); }

}  // namespace ops3d_reduce
