// Attention: kernel instantiations for element type _Float16.
#include "attention_kernels.h"

namespace ops3d_attention {

OPS3D_ATTENTION_TYPE(, _Float16)

}  // namespace ops3d_attention
