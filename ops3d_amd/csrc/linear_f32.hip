// Linear operators: kernel instantiations for element type float.
#include "linear_kernels.h"

namespace ops3d_linear {

template hipError_t forward<float>(const RowsArgs &, hipStream_t);
template hipError_t grad_x<float>(const RowsArgs &, hipStream_t);
template hipError_t grad_weight<float>(const WeightArgs &, int, bool, hipStream_t);
template hipError_t scale<float>(const void *, int64_t, const void *, void *, int64_t, int, hipStream_t);
template hipError_t keep_rows<float>(const void *, int64_t, void *, int64_t, int, const Groups &, hipStream_t);

}  // namespace ops3d_linear
