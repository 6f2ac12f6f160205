#include "group_norm.h"
#include "group_norm_host.h"

namespace amos {

// what a lane needs of its channels: h = (x - mean) rstd, z = h weight + bias
template <int VEC>
struct GnChannels {
  float mean[VEC], rstd[VEC], weight[VEC], bias[VEC];
  __device__ __forceinline__ GnChannels(const GnParams& p, int n, int c0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = c0 + i;
      const int64_t g = (int64_t)n * p.G + fast_div(c, p.by_cpg);
      mean[i] = p.mean[g];
      rstd[i] = p.rstd[g];
      weight[i] = p.weight ? load_any(p.weight, c, p.affine_dtype) : 1.f;
      bias[i] = p.bias ? load_any(p.bias, c, p.affine_dtype) : 0.f;
    }
  }
};

// ---- first launch: sums of d and d h over a chunk, by channel and (with the weights) by group -------
template <class XT, class YT, int VEC>
__global__ __launch_bounds__(kGnThreads) void amos_gn_gradient_partial(const GnParams p) {
  __shared__ float s1[kGnThreads * VEC], s2[kGnThreads * VEC];
  const GnTile w = gn_tile<VEC>(p, blockIdx.x);
  if (w.active) {
    const GnChannels<VEC> ch(p, w.n, w.c0 + w.col * VEC);
    const int64_t base = w.n * p.image + w.c0 + w.col * VEC;
    const typename XT::raw_t* const x = (const typename XT::raw_t*)p.x + base;
    const typename YT::raw_t* const dy = (const typename YT::raw_t*)p.dy + base;
    float a1[VEC], a2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) a1[i] = a2[i] = 0.f;
    for (int q = w.p0 + w.row; q < w.p1; q += p.rows) {
      float v[VEC], g[VEC];
      DenseVec<XT, VEC>::load(x + (int64_t)q * p.pixel, v);
      DenseVec<YT, VEC>::load(dy + (int64_t)q * p.pixel, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float h = (v[i] - ch.mean[i]) * ch.rstd[i];
        const float d = gn_act_gradient(g[i], h * ch.weight[i] + ch.bias[i], p.act);
        a1[i] += d;
        a2[i] += d * h;
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      s1[(w.row * p.cols + w.col) * VEC + i] = a1[i];
      s2[(w.row * p.cols + w.col) * VEC + i] = a2[i];
    }
  }
  __syncthreads();
  // ---- the pixel rows meet, in their order
  float* const cp = p.cpart + ((int64_t)blockIdx.x * p.C + w.c0) * 2;
  for (int c = threadIdx.x; c < w.width; c += kGnThreads) {
    float a = 0.f, b = 0.f;
    for (int r = 0; r < p.rows; ++r) {
      a += s1[r * p.cols * VEC + c];
      b += s2[r * p.cols * VEC + c];
    }
    cp[c * 2] = a;
    cp[c * 2 + 1] = b;
    const float weight = p.weight ? load_any(p.weight, w.c0 + c, p.affine_dtype) : 1.f;
    s1[c] = a * weight;   // (row 0: read above by this thread only)
    s2[c] = b * weight;
  }
  __syncthreads();
  const int team = gn_team(w.groups), t = threadIdx.x, lane = t & (team - 1), wide = w.width / w.groups;
  for (int g = t / team; g < w.groups; g += kGnThreads / team) {
    float a = 0.f, b = 0.f;
    for (int e = lane; e < wide; e += team) {
      a += s1[g * wide + e];
      b += s2[g * wide + e];
    }
    a = gn_team_sum(a, team);
    b = gn_team_sum(b, team);
    if (lane == 0) {
      const int slot = w.chunk * p.sub + (p.sub > 1 ? w.tile % p.sub : 0);
      float* at = p.part + (((int64_t)w.n * p.G + w.g0 + g) * p.slots + slot) * 2;
      at[0] = a;
      at[1] = b;
    }
  }
}

// dweight, dbias: sixteen channels a workgroup, sixteen rows of partial sums side by side
__device__ __forceinline__ void gn_coefficient_gradients(const GnParams& p, int block, float* s1, float* s2) {
  const int t = threadIdx.x, c = block * 16 + (t & 15), r0 = t >> 4;
  const int rows = p.N * p.chunks;
  float a = 0.f, b = 0.f;
  if (c < p.C) {
    const float* at = p.cpart + (int64_t)c * 2;
    for (int r = r0; r < rows; r += 16) {
      a += at[(int64_t)r * p.C * 2];
      b += at[(int64_t)r * p.C * 2 + 1];
    }
  }
  s1[t] = a;
  s2[t] = b;
  __syncthreads();
  if (t < 16 && c < p.C) {
    a = b = 0.f;
    for (int r = 0; r < 16; ++r) {
      a += s1[r * 16 + t];
      b += s2[r * 16 + t];
    }
    if (p.dbias) p.dbias[c] = a;
    if (p.dweight) p.dweight[c] = b;
  }
}

// ---- second launch: dx; behind the workgroups of the tiles those of dweight and dbias ---------------
template <class XT, class YT, int VEC>
__global__ __launch_bounds__(kGnThreads) void amos_gn_gradient_apply(const GnParams p) {
  __shared__ float s1[kGnThreads * VEC], s2[kGnThreads * VEC];   // by group of the tile: E[d weight], E[d weight h]
  if ((int)blockIdx.x >= p.N * p.chunks) {
    if (blockIdx.y == 0) gn_coefficient_gradients(p, (int)blockIdx.x - p.N * p.chunks, s1, s2);
    return;
  }
  const GnTile w = gn_tile<VEC>(p, blockIdx.x);
  {
    const int team = gn_team(w.groups), t = threadIdx.x, lane = t & (team - 1);
    const float share = 1.f / ((float)p.P * p.cpg);
    for (int g = t / team; g < w.groups; g += kGnThreads / team) {
      const float* at = p.part + ((int64_t)w.n * p.G + w.g0 + g) * p.slots * 2;
      float a = 0.f, b = 0.f;
      for (int e = lane; e < p.slots; e += team) {
        a += at[e * 2];
        b += at[e * 2 + 1];
      }
      a = gn_team_sum(a, team);
      b = gn_team_sum(b, team);
      if (lane == 0) {
        s1[g] = a * share;
        s2[g] = b * share;
      }
    }
  }
  __syncthreads();
  if (!w.active) return;
  const GnChannels<VEC> ch(p, w.n, w.c0 + w.col * VEC);
  float e1[VEC], e2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int g = fast_div(w.c0 + w.col * VEC + i, p.by_cpg) - w.g0;
    e1[i] = s1[g];
    e2[i] = s2[g];
  }
  const int64_t base = w.n * p.image + w.c0 + w.col * VEC;
  const typename XT::raw_t* const x = (const typename XT::raw_t*)p.x + base;
  const typename YT::raw_t* const dy = (const typename YT::raw_t*)p.dy + base;
  typename XT::raw_t* const dx = (typename XT::raw_t*)p.out + base;
  for (int q = w.p0 + w.row; q < w.p1; q += p.rows) {
    float v[VEC], g[VEC];
    DenseVec<XT, VEC>::load(x + (int64_t)q * p.pixel, v);
    DenseVec<YT, VEC>::load(dy + (int64_t)q * p.pixel, g);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float h = (v[i] - ch.mean[i]) * ch.rstd[i];
      const float d = gn_act_gradient(g[i], h * ch.weight[i] + ch.bias[i], p.act);
      v[i] = (d * ch.weight[i] - e1[i] - h * e2[i]) * ch.rstd[i];
    }
    DenseVec<XT, VEC>::store(dx + (int64_t)q * p.pixel, v);
  }
}

template <class XT, class YT, int VEC>
static void launch(const GnParams& p, hipStream_t stream) {
  const unsigned work = (unsigned)((int64_t)p.N * p.chunks);
  const unsigned more = p.dweight || p.dbias ? (unsigned)((p.C + 15) / 16) : 0;
  hipLaunchKernelGGL((amos_gn_gradient_partial<XT, YT, VEC>), dim3(work, (unsigned)p.tiles), dim3(kGnThreads), 0, stream, p);
  hipLaunchKernelGGL((amos_gn_gradient_apply<XT, YT, VEC>), dim3(work + more, (unsigned)p.tiles), dim3(kGnThreads), 0, stream, p);
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

static int run_gradient(const amos_group_norm_desc_t* d, const void* dy, const void* x, const void* weight, const void* bias, const float* mean,
                        const float* rstd, void* dx, float* dweight, float* dbias, void* workspace, size_t ws_bytes, hipStream_t stream) {
  GnParams p;
  GnPlan plan;
  int rc = gn_plan(d, {dy, x, dx}, weight, bias, p, plan);
  if (rc) return rc;
  if (!mean || !rstd) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  rc = gn_workspace(plan, p, true, workspace, ws_bytes);
  if (rc) return rc;
  p.x = x;
  p.dy = dy;
  p.out = dx;
  p.mean = (float*)mean;
  p.rstd = (float*)rstd;
  p.dweight = dweight;
  p.dbias = dbias;
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

int amos_group_norm_backward(const amos_group_norm_desc_t* desc, const void* dy, const void* x, const void* weight, const void* bias,
                             const float* mean, const float* rstd, void* dx, float* dweight, float* dbias, void* workspace, size_t ws_bytes,
                             void* stream) {
  return run_gradient(desc, dy, x, weight, bias, mean, rstd, dx, dweight, dbias, workspace, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
