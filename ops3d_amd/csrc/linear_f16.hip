// Linear operators: kernel instantiations for element type _Float16.
#include "linear_kernels.h"

namespace ops3d_linear {

template hipError_t forward<_Float16>(const RowsArgs &, hipStream_t);
template hipError_t grad_x<_Float16>(const RowsArgs &, hipStream_t);
template hipError_t grad_weight<_Float16>(const WeightArgs &, int, bool, hipStream_t);
template hipError_t scale<_Float16>(const void *, int64_t, const void *, void *, int64_t, int, hipStream_t);
template hipError_t keep_rows<_Float16>(const void *, int64_t, void *, int64_t, int, const Groups &, hipStream_t);

}  // namespace ops3d_linear
