#include "group_norm.h"
#include "group_norm_host.h"

namespace amos {

// ---- first launch: a chunk's (count, mean, squared deviations) for every group of the tile --------
template <class XT, int VEC>
__global__ __launch_bounds__(kGnThreads) void amos_gn_partial(const GnParams p) {
  __shared__ float smean[kGnThreads * VEC], sm2[kGnThreads * VEC];
  const GnTile w = gn_tile<VEC>(p, blockIdx.x);
  float mean[VEC], m2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) mean[i] = m2[i] = 0.f;
  if (w.active) {
    const typename XT::raw_t* x = (const typename XT::raw_t*)p.x + w.n * p.image + w.c0 + w.col * VEC;
    float cnt = 0.f;
    int q = w.p0 + w.row;
    constexpr int B = 4;
    // four pixels at a time: their own mean and deviations, joined to the running ones
    for (; q + (B - 1) * p.rows < w.p1; q += B * p.rows) {
      float v[B][VEC];
#pragma unroll
      for (int b = 0; b < B; ++b) DenseVec<XT, VEC>::load(x + (int64_t)(q + b * p.rows) * p.pixel, v[b]);
      const float share = (float)B / (cnt + B), both = cnt * share;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float s = 0.f, d2 = 0.f;
#pragma unroll
        for (int b = 0; b < B; ++b) s += v[b][i];
        s *= 1.f / B;
#pragma unroll
        for (int b = 0; b < B; ++b) d2 += (v[b][i] - s) * (v[b][i] - s);
        const float delta = s - mean[i];
        mean[i] += delta * share;
        m2[i] += d2 + delta * delta * both;
      }
      cnt += B;
    }
    for (; q < w.p1; q += p.rows) {
      float v[VEC];
      DenseVec<XT, VEC>::load(x + (int64_t)q * p.pixel, v);
      const float share = 1.f / (cnt + 1.f), both = cnt * share;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float delta = v[i] - mean[i];
        mean[i] += delta * share;
        m2[i] += delta * delta * both;
      }
      cnt += 1.f;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      smean[w.row * p.cols * VEC + w.col * VEC + i] = mean[i];
      sm2[w.row * p.cols * VEC + w.col * VEC + i] = m2[i];
    }
  }
  __syncthreads();
  // ---- the pixel rows and channels of a group meet: first their mean, then the deviations from it
  const int team = gn_team(w.groups), t = threadIdx.x, lane = t & (team - 1);
  const int span = w.p1 - w.p0, wide = w.width / w.groups;
  const int entries = p.rows * wide;
  for (int g = t / team; g < w.groups; g += kGnThreads / team) {   // (a team comes here whole)
    float s = 0.f;
    for (int e = lane; e < entries; e += team) {
      const int r = e / wide, c = g * wide + (e - r * wide);
      const int k = span > r ? (span - r + p.rows - 1) / p.rows : 0;   // pixels of this row of threads
      if (k > 0) s += (float)k * smean[r * p.cols * VEC + c];
    }
    const float total = (float)span * wide;
    const float m = gn_team_sum(s, team) / total;
    float d = 0.f;
    for (int e = lane; e < entries; e += team) {
      const int r = e / wide, c = g * wide + (e - r * wide);
      const int k = span > r ? (span - r + p.rows - 1) / p.rows : 0;
      if (k > 0) {
        const float off = smean[r * p.cols * VEC + c] - m;
        d += sm2[r * p.cols * VEC + c] + (float)k * off * off;
      }
    }
    d = gn_team_sum(d, team);
    if (lane == 0) {
      const int s_at = w.chunk * p.sub + (p.sub > 1 ? w.tile % p.sub : 0);
      float* at = p.part + (((int64_t)w.n * p.G + w.g0 + g) * p.slots + s_at) * 3;
      at[0] = total;
      at[1] = m;
      at[2] = d;
    }
  }
}

// the statistics of group `g` of image `n` from its slots, by a team; every thread of it gets them
__device__ __forceinline__ void gn_join(const GnParams& p, int n, int g, int lane, int team, float& mean, float& rstd) {
  const float* at = p.part + ((int64_t)n * p.G + g) * p.slots * 3;
  float s = 0.f;
  for (int e = lane; e < p.slots; e += team) s += at[e * 3] * at[e * 3 + 1];
  const float total = (float)p.P * p.cpg;
  mean = gn_team_sum(s, team) / total;
  float d = 0.f;
  for (int e = lane; e < p.slots; e += team) {
    const float off = at[e * 3 + 1] - mean;
    d += at[e * 3 + 2] + at[e * 3] * off * off;
  }
  const float var = gn_team_sum(d, team) / total;
  rstd = 1.f / sqrtf(var + p.eps);
}

// ---- second launch: normalise, scale, activate ----------------------------------------------------
template <class XT, class YT, int VEC>
__global__ __launch_bounds__(kGnThreads) void amos_gn_apply(const GnParams p) {
  __shared__ float smean[kGnThreads * VEC], srstd[kGnThreads * VEC];   // by group of the tile
  const GnTile w = gn_tile<VEC>(p, blockIdx.x);
  {
    const int team = gn_team(w.groups), t = threadIdx.x, lane = t & (team - 1), step = kGnThreads / team;
    for (int g = t / team; g < w.groups; g += step) {
      float mean, rstd;
      gn_join(p, w.n, w.g0 + g, lane, team, mean, rstd);
      if (lane == 0) {
        smean[g] = mean;
        srstd[g] = rstd;
        if (w.chunk == 0 && (p.sub == 1 || w.tile % p.sub == 0)) {
          if (p.mean) p.mean[(int64_t)w.n * p.G + w.g0 + g] = mean;
          if (p.rstd) p.rstd[(int64_t)w.n * p.G + w.g0 + g] = rstd;
        }
      }
    }
  }
  __syncthreads();
  if (!w.active) return;
  float m[VEC], a[VEC], b[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int c = w.c0 + w.col * VEC + i;
    const int g = fast_div(c, p.by_cpg) - w.g0;
    m[i] = smean[g];
    a[i] = srstd[g] * (p.weight ? load_any(p.weight, c, p.affine_dtype) : 1.f);
    b[i] = p.bias ? load_any(p.bias, c, p.affine_dtype) : 0.f;
  }
  const int64_t base = w.n * p.image + w.c0 + w.col * VEC;
  const typename XT::raw_t* const x = (const typename XT::raw_t*)p.x + base;
  typename YT::raw_t* const y = (typename YT::raw_t*)p.out + base;
  for (int q = w.p0 + w.row; q < w.p1; q += p.rows) {
    float v[VEC];
    DenseVec<XT, VEC>::load(x + (int64_t)q * p.pixel, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = gn_act((v[i] - m[i]) * a[i] + b[i], p.act);
    DenseVec<YT, VEC>::store(y + (int64_t)q * p.pixel, v);
  }
}

template <class XT, class YT, int VEC>
static void launch(const GnParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.N * p.chunks), (unsigned)p.tiles), block(kGnThreads);
  hipLaunchKernelGGL((amos_gn_partial<XT, VEC>), grid, block, 0, stream, p);
  hipLaunchKernelGGL((amos_gn_apply<XT, YT, VEC>), grid, block, 0, stream, p);
}
template <class XT, class YT>
static void pick_vec(const GnParams& p, int vec, hipStream_t stream) {
  if (vec == 8) launch<XT, YT, 8>(p, stream);
  else launch<XT, YT, 1>(p, stream);
}
template <class XT>
static void pick_out(const GnParams& p, int vec, int y_dtype, hipStream_t stream) {
  if (y_dtype == AMOS_F32) pick_vec<XT, TypeF32>(p, vec, stream);
  else if (y_dtype == AMOS_F16) pick_vec<XT, TypeF16>(p, vec, stream);
  else pick_vec<XT, TypeBF16>(p, vec, stream);
}

static int run_forward(const amos_group_norm_desc_t* d, const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                       void* workspace, size_t ws_bytes, hipStream_t stream) {
  GnParams p;
  GnPlan plan;
  int rc = gn_plan(d, {x, y}, weight, bias, p, plan);
  if (rc) return rc;
  rc = gn_workspace(plan, p, false, workspace, ws_bytes);
  if (rc) return rc;
  p.x = x;
  p.out = y;
  p.mean = mean;
  p.rstd = rstd;
  if (d->x_dtype == AMOS_F32) pick_out<TypeF32>(p, plan.vec, d->y_dtype, stream);
  else if (d->x_dtype == AMOS_F16) pick_out<TypeF16>(p, plan.vec, d->y_dtype, stream);
  else pick_out<TypeBF16>(p, plan.vec, d->y_dtype, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  return 0;
}

}  // namespace amos

using namespace amos;

extern "C" {

size_t amos_group_norm_workspace_bytes(const amos_group_norm_desc_t* desc, int gradient) {
  return gn_workspace_bytes(desc, gradient != 0);
}

int amos_group_norm(const amos_group_norm_desc_t* desc, const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                    void* workspace, size_t ws_bytes, void* stream) {
  return run_forward(desc, x, weight, bias, y, mean, rstd, workspace, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
