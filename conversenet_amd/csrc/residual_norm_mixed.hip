// residual_norm.h with a float32 residual stream and a 16-bit branch.
#include "residual_norm_kernels.h"

namespace cvn {
RnKernels rn_f32_bf16() { return {rn_launch_fwd<float, __bf16>, rn_launch_bwd<float, __bf16>}; }
RnKernels rn_f32_f16() { return {rn_launch_fwd<float, _Float16>, rn_launch_bwd<float, _Float16>}; }
}  // namespace cvn
