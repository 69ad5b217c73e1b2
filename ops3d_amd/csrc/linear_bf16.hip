// Linear operators: kernel instantiations for element type __bf16.
#include "linear_kernels.h"

namespace ops3d_linear {

template hipError_t forward<__bf16>(const RowsArgs &, hipStream_t);
template hipError_t grad_x<__bf16>(const RowsArgs &, hipStream_t);
template hipError_t grad_weight<__bf16>(const WeightArgs &, int, bool, hipStream_t);
template hipError_t scale<__bf16>(const void *, int64_t, const void *, void *, int64_t, int, hipStream_t);
template hipError_t keep_rows<__bf16>(const void *, int64_t, void *, int64_t, int, const Groups &, hipStream_t);

}  // namespace ops3d_linear
