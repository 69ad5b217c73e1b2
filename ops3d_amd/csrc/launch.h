// Launches of more blocks than one may have.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ops3d_launch {

// A launch holds less than 2^32 threads; more go in several, each a multiple of the XCDs' 8 blocks.  p.block0: blocks
// in launches before this one.
template <typename K, typename A> inline hipError_t launch(K kernel, int64_t grid, int threads, hipStream_t st, A p) {
  if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
  const int64_t most = 0xffffffff / threads & ~(int64_t)7;
  for (int64_t at = 0; at < grid; at += most) {
    p.block0 = (unsigned)at;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(grid - at < most ? grid - at : most)), dim3(threads), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ops3d_launch
