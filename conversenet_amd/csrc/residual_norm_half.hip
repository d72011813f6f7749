// residual_norm.h with a 16-bit residual stream.
#include "residual_norm_kernels.h"

namespace cvn {
RnKernels rn_bf16_bf16() { return {rn_launch_fwd<__bf16, __bf16>, rn_launch_bwd<__bf16, __bf16>}; }
RnKernels rn_f16_f16() { return {rn_launch_fwd<_Float16, _Float16>, rn_launch_bwd<_Float16, _Float16>}; }
}  // namespace cvn
