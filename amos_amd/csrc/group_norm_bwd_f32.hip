#include "group_norm_bwd_kernels.h"
namespace amos {
int group_norm_gradient_f32(const GnParams& p, const GnPlan& plan, hipStream_t stream) { return launch_gradient<TypeF32>(p, plan, stream); }
}  // namespace amos
