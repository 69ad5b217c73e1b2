// Walks over a table of consecutive segments of rows that only the device knows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ops3d_segments {

// Inclusive scans over a wave.
__device__ __forceinline__ int scan_add(int v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o);
    if ((int)(threadIdx.x & 63) >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ int scan_max(int v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o);
    if ((int)(threadIdx.x & 63) >= o) v = max(v, t);
  }
  return v;
}

// Segments of S rows: 0 the rows before the first entry, e + 1 those from entry e on, behind the last entry
// those up to S.  Entries count as the largest of themselves and those before them, held to [0, S].  One
// step of a walk over them, 64 at a time, segment j a lane; carry: the last upper bound, 0 before the first
// step.
struct Segment {
  int lower, upper;   // rows
};
__device__ __forceinline__ Segment segment_at(const int64_t *start, int count, int S, int j, int &carry) {
  int64_t v = j < count ? start[j] : (int64_t)S;
  v = v < 0 ? 0 : (v > S ? S : v);
  Segment s;
  s.upper = max(scan_max((int)v), carry);
  s.lower = __shfl_up(s.upper, 1);
  if ((threadIdx.x & 63) == 0) s.lower = carry;
  carry = __builtin_amdgcn_readlane(s.upper, 63);
  return s;
}

}  // namespace ops3d_segments
