#include "group_norm.h"
#include "group_norm_host.h"

namespace amos {

// ---- first launch: a chunk's (count, mean, squared deviations) for every group of the tile --------
// (no difference of large sums, whatever the mean is)
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
    // four pixels at a time: their own mean and deviations, joined to the running ones (delta times delta times `both` in this
    // order: in front of the first pixels `both` is 0 and delta the mean itself, whose square fp32 need not hold)
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
        m2[i] += d2 + delta * (delta * both);
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
        m2[i] += delta * (delta * both);
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
  const int each = span / p.rows, more = span - each * p.rows;   // pixels of a row of threads: each, one more in the first `more`
  const auto row_of = [&](int e) { return p.sub > 1 ? (e >= wide ? 1 : 0) : fast_div(e, p.by_cpg); };   // (tiles inside a group: at most two rows)
  for (int g = t / team; g < w.groups; g += kGnThreads / team) {   // (a team comes here whole)
    float s = 0.f;
#pragma unroll 4
    for (int e = lane; e < entries; e += team) {
      const int r = row_of(e), c = g * wide + (e - r * wide);
      s += (float)(each + (r < more)) * smean[r * p.cols * VEC + c];   // (a row without pixels holds zeros)
    }
    const float total = (float)span * wide;
    const float m = gn_team_sum(s, team) / total;
    float d = 0.f;
#pragma unroll 4
    for (int e = lane; e < entries; e += team) {
      const int r = row_of(e), c = g * wide + (e - r * wide);
      const float off = smean[r * p.cols * VEC + c] - m;
      d += sm2[r * p.cols * VEC + c] + (float)(each + (r < more)) * off * off;
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
  rstd = gn_rstd(var, p.eps);
}

// ---- second launch: normalise, scale, activate ----------------------------------------------------
template <class XT, class YT, int VEC, bool SILU>
__global__ __launch_bounds__(kGnThreads) void amos_gn_apply(const GnParams p) {
  __shared__ float smean[kGnThreads * VEC], srstd[kGnThreads * VEC];   // by group of the tile
  const GnTile w = gn_tile<VEC>(p, blockIdx.x);
  float m[VEC], a[VEC], b[VEC];
  load_run_any<VEC>(p.weight, w.c0 + (w.active ? w.col * VEC : 0), p.affine_dtype, 1.f, a);
  load_run_any<VEC>(p.bias, w.c0 + (w.active ? w.col * VEC : 0), p.affine_dtype, 0.f, b);
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
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int g = fast_div(w.c0 + w.col * VEC + i, p.by_cpg) - w.g0;
    m[i] = smean[g];
    a[i] *= srstd[g];
  }
  const int64_t base = w.n * p.image + w.c0 + w.col * VEC;
  const typename XT::raw_t* const x = (const typename XT::raw_t*)p.x + base;
  typename YT::raw_t* const y = (typename YT::raw_t*)p.out + base;
  constexpr int B = 4;
  int q = w.p0 + w.row;
  for (; q + (B - 1) * p.rows < w.p1; q += B * p.rows) {   // four pixels in flight
    typename DenseVec<XT, VEC>::vec_t raw[B];
#pragma unroll
    for (int u = 0; u < B; ++u) raw[u] = DenseVec<XT, VEC>::read(x + (int64_t)(q + u * p.rows) * p.pixel);
#pragma unroll
    for (int u = 0; u < B; ++u) {
      float v[VEC];
      DenseVec<XT, VEC>::widen(raw[u], v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = gn_act<SILU>((v[i] - m[i]) * a[i] + b[i], p.low);
      DenseVec<YT, VEC>::store(y + (int64_t)(q + u * p.rows) * p.pixel, v);
    }
  }
  for (; q < w.p1; q += p.rows) {
    float v[VEC];
    DenseVec<XT, VEC>::load(x + (int64_t)q * p.pixel, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = gn_act<SILU>((v[i] - m[i]) * a[i] + b[i], p.low);
    DenseVec<YT, VEC>::store(y + (int64_t)q * p.pixel, v);
  }
}

// ---- one launch: a slab of whole groups stays in registers between the sums and the output -----------
// One pass over memory.  A thread holds R vectors of 16 bytes (all its loads are in flight together); mean, then the
// squared deviations from it, from the registers.  32 x 56 x 56 x 256 bf16 + silu (103 MB): 26 us = 4.0 TB/s, two launches
// 50 us; what a copy of as many bytes does not have is the pause between a compute unit's reads and its writes (its one
// workgroup waits for the sums).  1 x 7 x 7 x 512 fp32: 5 us, a chain of a load, two sums over LDS and a store.
template <class XT, int VEC, int R, bool UNI, bool SILU>
__global__ __launch_bounds__(1024) void amos_gn_held(const GnParams p) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  typedef DenseVec<XT, VEC> V;
  const GnSlab w = gn_slab(p, VEC);
  const int per = UNI ? p.cols : p.cols * VEC;
  float* const total = lds + p.rows * per;
  const typename XT::raw_t* const x = (const typename XT::raw_t*)p.x + w.n * p.image + w.c;
  typename V::vec_t raw[R];
  if (w.active) {
#pragma unroll
    for (int r = 0; r < R; ++r) {   // (pixels past the end: the last one again, left out of the sums)
      if (r * p.rows >= p.P) break;
      const int q = w.row + r * p.rows;
      raw[r] = V::read(x + (int64_t)(q < p.P ? q : p.P - 1) * p.pixel);
    }
  }
  float gamma[VEC], beta[VEC];
  load_run_any<VEC>(p.weight, w.active ? w.c : w.c0, p.affine_dtype, 1.f, gamma);
  load_run_any<VEC>(p.bias, w.active ? w.c : w.c0, p.affine_dtype, 0.f, beta);
  constexpr int S = UNI ? 1 : VEC;   // sums a thread keeps
  float s[S], mean[S], rstd[S];
  int group[S];
#pragma unroll
  for (int i = 0; i < S; ++i) group[i] = w.active ? fast_div(w.c + i, p.by_cpg) - w.g0 : 0;
  const float count = (float)p.P * p.cpg;   // (divided by, not multiplied with its inverse: equal values have their own mean)
#pragma unroll
  for (int i = 0; i < S; ++i) s[i] = 0.f;
  if (w.active) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[VEC];
      V::widen(raw[r], v);
      if (w.row + r * p.rows < p.P) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[UNI ? 0 : i] += v[i];
      }
    }
  }
  gn_group_sums<VEC, UNI>(p, w, s, lds, total, [&](float sum) { return sum / count; });
#pragma unroll
  for (int i = 0; i < S; ++i) {
    mean[i] = total[group[i]];
    s[i] = 0.f;
  }
  if (w.active) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[VEC];
      V::widen(raw[r], v);
      if (w.row + r * p.rows < p.P) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = v[i] - mean[UNI ? 0 : i];
          s[UNI ? 0 : i] += d * d;
        }
      }
    }
  }
  gn_group_sums<VEC, UNI>(p, w, s, lds, total + w.groups, [&](float sum) { return gn_rstd(sum / count, p.eps); });
#pragma unroll
  for (int i = 0; i < S; ++i) rstd[i] = total[w.groups + group[i]];
  if (!w.active) return;
  if (w.row == 0) {   // a group's first lane and channel
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if ((w.g0 + group[i]) * p.cpg == w.c + i) {
        if (p.mean) p.mean[(int64_t)w.n * p.G + w.g0 + group[i]] = mean[i];
        if (p.rstd) p.rstd[(int64_t)w.n * p.G + w.g0 + group[i]] = rstd[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) gamma[i] *= rstd[UNI ? 0 : i];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int q = w.row + r * p.rows;
    if (q >= p.P) break;
    float v[VEC];
    V::widen(raw[r], v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = gn_act<SILU>((v[i] - mean[UNI ? 0 : i]) * gamma[i] + beta[i], p.low);
    store_run_any<VEC>(p.out, w.n * p.image + w.c + (int64_t)q * p.pixel, p.y_dtype, v);
  }
}

template <class XT, int VEC, bool UNI, bool SILU>
static void launch_held(const GnParams& p, const GnPlan& plan, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.N * p.tiles)), block((unsigned)plan.threads);
  if (plan.held <= 4) hipLaunchKernelGGL((amos_gn_held<XT, VEC, 4, UNI, SILU>), grid, block, plan.lds, stream, p);
  else hipLaunchKernelGGL((amos_gn_held<XT, VEC, kGnHeldForward, UNI, SILU>), grid, block, plan.lds, stream, p);
}
template <class XT, bool SILU>
static void pick_held(const GnParams& p, const GnPlan& plan, hipStream_t stream) {
  if constexpr (XT::ES == 2) {
    if (plan.vec == 8) return plan.uni ? launch_held<XT, 8, true, SILU>(p, plan, stream) : launch_held<XT, 8, false, SILU>(p, plan, stream);
  }
  if (plan.vec == 4) return plan.uni ? launch_held<XT, 4, true, SILU>(p, plan, stream) : launch_held<XT, 4, false, SILU>(p, plan, stream);
  launch_held<XT, 1, true, SILU>(p, plan, stream);
}

template <class XT, class YT, int VEC>
static void launch(const GnParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.N * p.chunks), (unsigned)p.tiles), block(kGnThreads);
  hipLaunchKernelGGL((amos_gn_partial<XT, VEC>), grid, block, 0, stream, p);
  if (p.act == AMOS_ACT_SILU) hipLaunchKernelGGL((amos_gn_apply<XT, YT, VEC, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((amos_gn_apply<XT, YT, VEC, false>), grid, block, 0, stream, p);
}
template <class XT, class YT>
static void pick_vec(const GnParams& p, int vec, hipStream_t stream) {
  constexpr int WIDE = XT::ES == 4 || YT::ES == 4 ? 4 : 8;   // 16 bytes of the wider type
  if (vec == WIDE) launch<XT, YT, WIDE>(p, stream);
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
  if (!d) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  int rc = gn_check(d, {{x, d->x_dtype}, {y, d->y_dtype}}, weight, bias, {mean, rstd}, p);
  if (rc == 0) rc = gn_choose(d, false, p, plan);
  if (rc == 0) rc = gn_workspace(plan, p, workspace, ws_bytes);
  if (rc) return rc;
  p.x = x;
  p.out = y;
  p.mean = mean;
  p.rstd = rstd;
  if (plan.held) {
    const bool silu = p.act == AMOS_ACT_SILU;
    if (d->x_dtype == AMOS_F32) silu ? pick_held<TypeF32, true>(p, plan, stream) : pick_held<TypeF32, false>(p, plan, stream);
    else if (d->x_dtype == AMOS_F16) silu ? pick_held<TypeF16, true>(p, plan, stream) : pick_held<TypeF16, false>(p, plan, stream);
    else silu ? pick_held<TypeBF16, true>(p, plan, stream) : pick_held<TypeBF16, false>(p, plan, stream);
  } else if (d->x_dtype == AMOS_F32) {
    pick_out<TypeF32>(p, plan.vec, d->y_dtype, stream);
  } else if (d->x_dtype == AMOS_F16) {
    pick_out<TypeF16>(p, plan.vec, d->y_dtype, stream);
  } else {
    pick_out<TypeBF16>(p, plan.vec, d->y_dtype, stream);
  }
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
