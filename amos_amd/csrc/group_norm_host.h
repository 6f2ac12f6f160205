// Argument checks and the plan (tiles, chunks, workspace) of the group norm launches.
#pragma once
#include <string.h>

#include <initializer_list>

#include "group_norm.h"
#include "mapper.h"

namespace amos {

inline int gn_tiles(const amos_group_norm_desc_t* d, int vec, GnParams& p, GnPlan& plan) {
  const int64_t most = (int64_t)kGnThreads * vec;   // channels a workgroup can lay side by side
  const int64_t C = d->C, cpg = C / d->groups;
  int64_t ct, tiles, sub = 1;
  if (C % vec) return 1;
  if (C <= most) {
    ct = C;
    tiles = 1;
  } else if (cpg <= most) {            // whole groups, and whole vectors
    int64_t unit = 1;
    while (unit * cpg % vec) ++unit;
    const int64_t per_tile = most / cpg / unit * unit;
    if (per_tile == 0) return 1;
    ct = per_tile * cpg;
    tiles = (d->groups + per_tile - 1) / per_tile;
  } else {                             // several tiles a group
    if (cpg % vec) return 1;
    sub = (cpg + most - 1) / most;
    ct = ((cpg + sub - 1) / sub + vec - 1) / vec * vec;
    sub = (cpg + ct - 1) / ct;
    tiles = d->groups * sub;
  }
  if (tiles > 65535) return set_error(AMOS_ERR_UNSUPPORTED, "group norm of %lld channels in %d groups", (long long)C, d->groups);
  plan.vec = vec;
  p.ct = (int)ct;
  p.tiles = (int)tiles;
  p.sub = (int)sub;
  p.cols = (int)((ct + vec - 1) / vec);
  p.rows = kGnThreads / p.cols;
  // chunks: some 2048 workgroups, each thread at least eight pixels, at most 128 partial results to join
  const int64_t P = p.P;
  int64_t chunks = 2048 / (d->N * tiles);
  chunks = chunks < 1 ? 1 : chunks > 128 ? 128 : chunks;
  int64_t chunk = (P + chunks - 1) / chunks;
  if (chunk < 8 * p.rows) chunk = 8 * p.rows;
  if (chunk > P) chunk = P;
  p.chunk = (int)chunk;
  p.chunks = (int)((P + chunk - 1) / chunk);
  if ((int64_t)p.N * p.chunks + C >= (int64_t)1 << 31) return set_error(AMOS_ERR_UNSUPPORTED, "group norm of %d images", p.N);
  p.slots = p.chunks * p.sub;
  p.by_cols = make_fast_div((uint32_t)p.cols);
  p.by_cpg = make_fast_div((uint32_t)p.cpg);
  plan.part_floats = (int64_t)p.N * p.G * p.slots * 3;
  plan.cpart_floats = (int64_t)p.N * p.chunks * p.C * 2;
  return 0;
}

inline int gn_plan(const amos_group_norm_desc_t* d, std::initializer_list<const void*> tensors, const void* weight, const void* bias, GnParams& p,
                   GnPlan& plan) {
  if (!d) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  for (const void* t : tensors)
    if (!t) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  memset(&p, 0, sizeof(p));
  if (d->N < 1 || d->C < 1 || d->D < 1 || d->H < 1 || d->W < 1)
    return set_error(AMOS_ERR_BAD_ARG, "group norm of extents N %lld, D %lld, H %lld, W %lld, C %lld", (long long)d->N, (long long)d->D,
                     (long long)d->H, (long long)d->W, (long long)d->C);
  if (d->groups < 1 || d->C % d->groups) return set_error(AMOS_ERR_BAD_ARG, "group norm: %lld channels in %d groups", (long long)d->C, d->groups);
  const int64_t lim = (int64_t)1 << 28;
  if (d->N >= lim || d->C >= lim || d->D >= lim || d->H >= lim || d->W >= lim || d->D * d->H >= lim || d->D * d->H * d->W >= lim)
    return set_error(AMOS_ERR_UNSUPPORTED, "group norm: images, channels or pixels of an image beyond 2^28");
  if (d->layout != AMOS_LAYOUT_NHWC && d->layout != AMOS_LAYOUT_HWNC)
    return set_error(AMOS_ERR_UNSUPPORTED, "group norm: layout %d (channels-last layouts only)", d->layout);
  if (d->activation != AMOS_ACT_NONE && d->activation != AMOS_ACT_RELU && d->activation != AMOS_ACT_SILU)
    return set_error(AMOS_ERR_UNSUPPORTED, "group norm: activation %d", d->activation);
  if (!is_dense_dtype(d->x_dtype) || !is_dense_dtype(d->y_dtype) || ((weight || bias) && !is_dense_dtype(d->affine_dtype)))
    return set_error(AMOS_ERR_UNSUPPORTED, "group norm: dtypes %d, %d, %d (fp32, fp16 or bf16)", d->x_dtype, d->y_dtype, d->affine_dtype);
  if (!(d->eps >= 0.f) || d->eps > 3e38f) return set_error(AMOS_ERR_BAD_ARG, "group norm: eps %g", (double)d->eps);
  p.N = (int)d->N;
  p.P = (int)(d->D * d->H * d->W);
  p.C = (int)d->C;
  p.G = d->groups;
  p.cpg = p.C / p.G;
  p.image = d->layout == AMOS_LAYOUT_NHWC ? (int64_t)p.P * p.C : p.C;
  p.pixel = d->layout == AMOS_LAYOUT_NHWC ? p.C : (int64_t)p.N * p.C;
  p.eps = d->eps;
  p.act = d->activation;
  p.affine_dtype = d->affine_dtype;
  p.weight = weight;
  p.bias = bias;
  const int es = dense_size(d->x_dtype) < dense_size(d->y_dtype) ? dense_size(d->x_dtype) : dense_size(d->y_dtype);
  bool wide = true;
  for (const void* t : tensors) {
    if ((uintptr_t)t & (es - 1)) return set_error(AMOS_ERR_BAD_ARG, "group norm: misaligned tensor");
    wide = wide && ((uintptr_t)t & 15) == 0;
  }
  int rc = wide ? gn_tiles(d, 8, p, plan) : 1;
  if (rc == 1) rc = gn_tiles(d, 1, p, plan);
  return rc;
}

inline size_t gn_plan_bytes(const GnPlan& plan, bool gradient) {
  return (size_t)(plan.part_floats + (gradient ? plan.cpart_floats : 0)) * sizeof(float);
}
// enough for the vector kernels and for the element-wise ones (the choice goes by the pointers)
inline size_t gn_workspace_bytes(const amos_group_norm_desc_t* d, bool gradient) {
  GnParams p;
  GnPlan plan;
  if (gn_plan(d, {}, nullptr, nullptr, p, plan)) return 0;
  size_t need = gn_plan_bytes(plan, gradient);
  if (plan.vec != 1 && gn_tiles(d, 1, p, plan) == 0) {
    const size_t other = gn_plan_bytes(plan, gradient);
    need = other > need ? other : need;
  }
  return need;
}

inline int gn_workspace(const GnPlan& plan, GnParams& p, bool gradient, void* workspace, size_t ws_bytes) {
  const size_t need = gn_plan_bytes(plan, gradient);
  if (!workspace || ws_bytes < need || ((uintptr_t)workspace & 3))
    return set_error(AMOS_ERR_WORKSPACE, "group norm: %zu bytes of workspace wanted (amos_group_norm_workspace_bytes)", need);
  p.part = (float*)workspace;
  p.cpart = p.part + plan.part_floats;
  return 0;
}

}  // namespace amos
