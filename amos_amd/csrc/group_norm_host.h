// Argument checks and the plan (kernel, tiles, chunks, workspace) of the group norm launches.
#pragma once
#include <string.h>

#include <initializer_list>

#include "group_norm.h"
#include "mapper.h"

namespace amos {

constexpr int kGnHeldForward = 16, kGnHeldGradient = 6;   // vectors a thread of the one-launch kernels holds at most
constexpr int kGnHeldThreads = 1024;
constexpr int64_t kGnGridThreads = (int64_t)1 << 32;   // a grid's first extent has fewer

// The one-launch plan: as many groups a slab as bring a pixel's piece to 64 bytes (half a memory line), where
// a workgroup's registers hold that much.
inline bool gn_plan_held(const amos_group_norm_desc_t* d, bool gradient, int vec, GnParams& p, GnPlan& plan) {
  const int es = dense_size(d->x_dtype), most = gradient ? kGnHeldGradient : kGnHeldForward;
  int64_t unit = p.cpg;
  while (unit % vec) unit += p.cpg;   // whole groups and whole vectors
  if (p.C % unit) return false;
  const auto fits = [&](int64_t c) {
    const int64_t cols = c / vec;
    if (cols > kGnHeldThreads) return false;
    const int64_t rows = kGnHeldThreads / cols;
    return (p.P + rows - 1) / rows <= most;
  };
  if (!fits(unit)) return false;
  int64_t ct = unit;
  for (int64_t k = 2; ct * es < 64 && k * unit <= p.C && k <= 64; ++k)
    if (p.C % (k * unit) == 0 && fits(k * unit)) ct = k * unit;
  // (measured on 32 x 56 x 56 x 256 bf16: pieces of 16 bytes 82 us where two launches over whole rows take half)
  if (ct * es < 64 && ct < p.C && (int64_t)p.N * p.P * p.C * es > (int64_t)4 << 20) return false;
  p.ct = (int)ct;
  p.tiles = (int)(p.C / ct);
  p.sub = p.chunks = 1;
  p.chunk = p.P;
  p.cols = (int)(ct / vec);
  // some four vectors a thread (two for the gradient, which holds two tensors) before there are more threads
  int rows = kGnHeldThreads / p.cols;
  const int each = gradient ? 2 : 4;
  if ((p.P + each - 1) / each < rows) rows = (p.P + each - 1) / each;
  p.rows = rows;
  plan.vec = vec;
  plan.uni = p.cpg % vec == 0;
  plan.held = (p.P + p.rows - 1) / p.rows;
  plan.threads = (p.rows * p.cols + 63) / 64 * 64;
  const int per = plan.uni && !gradient ? p.cols : (int)ct;   // values of a row of threads that meet in LDS
  p.by_epg = make_fast_div((uint32_t)(per / (p.ct / p.cpg)));
  p.by_cols = make_fast_div((uint32_t)p.cols);
  p.by_cpg = make_fast_div((uint32_t)p.cpg);
  plan.lds = (p.rows * per * (gradient ? 2 : 1) + 2 * (p.ct / p.cpg)) * (int)sizeof(float);
  plan.part_floats = 0;
  plan.cpart_floats = gradient && p.N > 1 ? (int64_t)p.N * p.C * 2 : 0;   // the images' shares of dweight and dbias
  return plan.lds <= 96 * 1024 && p.N * (p.C / ct) * plan.threads < kGnGridThreads && (d->C / 16 + 1) * 256 < kGnGridThreads;
}

// The two-launch plan; 1: this vector length does not divide the tiles
inline int gn_plan_tiles(const amos_group_norm_desc_t* d, bool gradient, int vec, GnParams& p, GnPlan& plan) {
  const int64_t most = (int64_t)kGnThreads * vec;   // channels a workgroup can lay side by side
  const int64_t C = d->C, cpg = C / d->groups, P = p.P;
  if (C % vec) return 1;
  // chunks: some 1024 workgroups, each thread at least four pixels, at most 128 partial results to join
  const auto lay = [&](int64_t ct, int64_t tiles) {
    p.ct = (int)ct;
    p.tiles = (int)tiles;
    p.cols = (int)((ct + vec - 1) / vec);
    p.rows = kGnThreads / p.cols;
    int64_t chunks = 1024 / (d->N * tiles);
    chunks = chunks < 1 ? 1 : chunks > 128 ? 128 : chunks;
    int64_t chunk = (P + chunks - 1) / chunks;
    if (chunk < 4 * p.rows) chunk = 4 * p.rows;
    if (chunk > P) chunk = P;
    p.chunk = (int)chunk;
    p.chunks = (int)((P + chunk - 1) / chunk);
    return p.N * tiles * p.chunks;   // workgroups
  };
  int64_t sub = 1;
  if (cpg <= most) {            // tiles of whole groups, and whole vectors
    int64_t unit = 1;
    while (unit * cpg % vec) ++unit;
    const auto tiles_of = [&](int64_t per_tile) { return (d->groups + per_tile - 1) / per_tile; };
    int64_t per_tile = C <= most ? d->groups : most / cpg / unit * unit;
    if (per_tile == 0) return 1;
    if (tiles_of(per_tile) > 65535) return set_error(AMOS_ERR_UNSUPPORTED, "group norm of %lld channels in %d groups", (long long)C, d->groups);
    int64_t now = lay(per_tile * cpg, tiles_of(per_tile));
    // few images: narrower tiles, down to a memory line of a pixel, as long as that makes more workgroups (each joins the
    // partial results of fewer groups then, too)
    while (now < 1024) {
      const int64_t next = (per_tile / 2 + unit - 1) / unit * unit;
      if (next == 0 || next >= per_tile || next * cpg * dense_size(d->x_dtype) < 128) break;
      const int64_t then = lay(next * cpg, tiles_of(next));
      if (then <= now) {
        lay(per_tile * cpg, tiles_of(per_tile));
        break;
      }
      now = then;
      per_tile = next;
    }
  } else {                      // several tiles a group
    if (cpg % vec) return 1;
    sub = (cpg + most - 1) / most;
    const int64_t ct = ((cpg + sub - 1) / sub + vec - 1) / vec * vec;
    sub = (cpg + ct - 1) / ct;
    if (d->groups * sub > 65535) return set_error(AMOS_ERR_UNSUPPORTED, "group norm of %lld channels in %d groups", (long long)C, d->groups);
    lay(ct, d->groups * sub);
  }
  plan.vec = vec;
  plan.held = 0;
  p.sub = (int)sub;
  if (((int64_t)p.N * p.chunks + C / 16 + 1) * kGnThreads >= kGnGridThreads) return set_error(AMOS_ERR_UNSUPPORTED, "group norm of %d images", p.N);
  p.slots = p.chunks * p.sub;
  p.by_cols = make_fast_div((uint32_t)p.cols);
  p.by_cpg = make_fast_div((uint32_t)p.cpg);
  plan.part_floats = (int64_t)p.N * p.G * p.slots * (gradient ? 2 : 3);
  plan.cpart_floats = gradient ? (int64_t)p.N * p.chunks * p.C * 2 : 0;
  return 0;
}

inline int gn_choose(const amos_group_norm_desc_t* d, bool gradient, GnParams& p, GnPlan& plan) {
  const int vec = d->x_dtype == AMOS_F32 || d->y_dtype == AMOS_F32 ? 4 : 8;   // 16 bytes of the wider type
  const bool divides = d->C % vec == 0;
  if (gn_plan_held(d, gradient, divides ? vec : 1, p, plan)) return 0;
  int rc = divides ? gn_plan_tiles(d, gradient, vec, p, plan) : 1;
  if (rc == 1) rc = gn_plan_tiles(d, gradient, 1, p, plan);
  return rc;
}

struct GnTensor {
  const void* at;
  int dtype;
};
// `tensors`: the dense ones; `vectors`: fp32 statistics and gradients, or null
inline int gn_check(const amos_group_norm_desc_t* d, std::initializer_list<GnTensor> tensors, const void* weight, const void* bias,
                    std::initializer_list<const void*> vectors, GnParams& p) {
  if (!d) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  for (const GnTensor& t : tensors)
    if (!t.at) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  memset(&p, 0, sizeof(p));
  if (d->N < 1 || d->C < 1 || d->D < 1 || d->H < 1 || d->W < 1)
    return set_error(AMOS_ERR_BAD_ARG, "group norm of extents N %lld, D %lld, H %lld, W %lld, C %lld", (long long)d->N, (long long)d->D,
                     (long long)d->H, (long long)d->W, (long long)d->C);
  if (d->groups < 1 || d->C % d->groups) return set_error(AMOS_ERR_BAD_ARG, "group norm: %lld channels in %d groups", (long long)d->C, d->groups);
  const int64_t lim = (int64_t)1 << 28;
  if (d->N >= lim || d->C >= lim || d->D >= lim || d->H >= lim || d->W >= lim || d->D * d->H >= lim || d->D * d->H * d->W >= lim)
    return set_error(AMOS_ERR_UNSUPPORTED, "group norm: images, channels or pixels of an image beyond 2^28");
  if (d->N * (d->D * d->H * d->W) >= ((int64_t)1 << 40) / d->C)
    return set_error(AMOS_ERR_UNSUPPORTED, "group norm: a tensor of 2^40 elements and more");
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
  p.low = d->activation == AMOS_ACT_RELU ? 0.f : __builtin_nanf("");
  p.affine_dtype = d->affine_dtype;
  p.y_dtype = d->y_dtype;
  p.weight = weight;
  p.bias = bias;
  for (const GnTensor& t : tensors)
    if ((uintptr_t)t.at & (dense_size(t.dtype) - 1)) return set_error(AMOS_ERR_BAD_ARG, "group norm: misaligned tensor");
  for (const void* t : {weight, bias})
    if (t && ((uintptr_t)t & (dense_size(d->affine_dtype) - 1))) return set_error(AMOS_ERR_BAD_ARG, "group norm: misaligned weight or bias");
  for (const void* t : vectors)
    if ((uintptr_t)t & 3) return set_error(AMOS_ERR_BAD_ARG, "group norm: misaligned statistics or gradients of the coefficients");
  return 0;
}

inline size_t gn_plan_bytes(const GnPlan& plan) { return (size_t)((plan.part_floats + 1) / 2 * 2 + plan.cpart_floats) * sizeof(float); }
inline size_t gn_workspace_bytes(const amos_group_norm_desc_t* d, bool gradient) {
  GnParams p;
  GnPlan plan;
  if (gn_check(d, {}, nullptr, nullptr, {}, p) || gn_choose(d, gradient, p, plan)) return 0;
  return gn_plan_bytes(plan);
}

inline int gn_workspace(const GnPlan& plan, GnParams& p, void* workspace, size_t ws_bytes) {
  const size_t need = gn_plan_bytes(plan);
  if (need && (!workspace || ws_bytes < need || ((uintptr_t)workspace & 7)))
    return set_error(AMOS_ERR_WORKSPACE, "group norm: %zu bytes of workspace wanted (amos_group_norm_workspace_bytes)", need);
  p.part = (float*)workspace;
  p.cpart = p.part + (plan.part_floats + 1) / 2 * 2;
  return 0;
}

}  // namespace amos
