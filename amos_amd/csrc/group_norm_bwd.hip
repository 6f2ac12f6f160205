#include "group_norm.h"
#include "group_norm_host.h"

namespace amos {

int group_norm_gradient_f32(const GnParams& p, const GnPlan& plan, hipStream_t stream);
int group_norm_gradient_f16(const GnParams& p, const GnPlan& plan, hipStream_t stream);
int group_norm_gradient_bf16(const GnParams& p, const GnPlan& plan, hipStream_t stream);

static int run_gradient(const amos_group_norm_desc_t* d, const void* dy, const void* x, const void* weight, const void* bias, const float* mean,
                        const float* rstd, void* dx, float* dweight, float* dbias, void* workspace, size_t ws_bytes, hipStream_t stream) {
  GnParams p;
  GnPlan plan;
  if (!d) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  int rc = gn_check(d, {{dy, d->y_dtype}, {x, d->x_dtype}, {dx, d->x_dtype}}, weight, bias, {mean, rstd, dweight, dbias}, p);
  if (rc) return rc;
  if (!mean || !rstd) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  rc = gn_choose(d, true, p, plan);
  if (rc == 0) rc = gn_workspace(plan, p, workspace, ws_bytes);
  if (rc) return rc;
  p.x = x;
  p.dy = dy;
  p.out = dx;
  p.mean = (float*)mean;
  p.rstd = (float*)rstd;
  p.dweight = dweight;
  p.dbias = dbias;
  if (d->x_dtype == AMOS_F32) rc = group_norm_gradient_f32(p, plan, stream);
  else if (d->x_dtype == AMOS_F16) rc = group_norm_gradient_f16(p, plan, stream);
  else rc = group_norm_gradient_bf16(p, plan, stream);
  if (rc) return rc;
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  return 0;
}

}  // namespace amos

using namespace amos;

extern "C" {

int amos_group_norm_backward(const amos_group_norm_desc_t* desc, const void* dy, const void* x, const void* weight, const void* bias,
                             const float* mean, const float* rstd, void* dx, float* dweight, float* dbias, void* workspace, size_t ws_bytes,
                             void* stream) {
  return run_gradient(desc, dy, x, weight, bias, mean, rstd, dx, dweight, dbias, workspace, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
