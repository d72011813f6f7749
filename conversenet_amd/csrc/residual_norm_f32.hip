// residual_norm.h with a float32 residual stream.
#include "residual_norm_kernels.h"

namespace cvn {
RnKernels rn_f32_f32() { return {rn_launch_fwd<float, float>, rn_launch_bwd<float, float>}; }
}  // namespace cvn
