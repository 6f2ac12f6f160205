#include "group_norm_bwd_kernels.h"
namespace amos {
int group_norm_gradient_bf16(const GnParams& p, const GnPlan& plan, hipStream_t stream) { return launch_gradient<TypeBF16>(p, plan, stream); }
}  // namespace amos
