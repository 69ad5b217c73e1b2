// Attention: kernel instantiations for element type __bf16.
#include "attention_kernels.h"

namespace ops3d_attention {

OPS3D_ATTENTION_TYPE(, __bf16)

}  // namespace ops3d_attention
