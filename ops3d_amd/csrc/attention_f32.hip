// Attention: kernel instantiations for element type float.
#include "attention_kernels.h"

namespace ops3d_attention {

OPS3D_ATTENTION_TYPE(, float)

}  // namespace ops3d_attention
