// Kernels of the group norm gradient; one translation unit for each type of x (group_norm_bwd_*.hip).
#pragma once
#include "group_norm.h"
#include "group_norm_host.h"
#include "lds_limit.h"

namespace amos {

// What a lane needs of its channels.  With t = x - mean (a difference, not folded into a constant: the mean may be large)
//   z = t a + bias, a = rstd weight;  sums of d and of d t (times rstd: d h) are kept, and
//   dx = d a - t rstd^2 E[d weight h] - rstd E[d weight] = d a - t k2 - k1:
// the launches are bound by their arithmetic as much as by memory, and each element takes two operations fewer.
template <int VEC>
struct GnChannels {
  float mean[VEC], rstd[VEC], a[VEC], bias[VEC];
  __device__ __forceinline__ GnChannels(const GnParams& p, int n, int c0) {
    load_run_any<VEC>(p.weight, c0, p.affine_dtype, 1.f, a);
    load_run_any<VEC>(p.bias, c0, p.affine_dtype, 0.f, bias);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int64_t g = (int64_t)n * p.G + fast_div(c0 + i, p.by_cpg);
      mean[i] = p.mean[g];
      rstd[i] = p.rstd[g];
      a[i] *= rstd[i];
    }
  }
  // d = dy act'(z) of channel i; t: x - mean
  template <bool SILU>
  __device__ __forceinline__ float d(int i, float t, float dy, float low) const {
    return gn_act_gradient<SILU>(dy, t * a[i] + bias[i], low);
  }
};

// 32 x 56 x 56 x 256 bf16 (154 MB in and out): 25 + 28 us with inputs from memory, 21 + 28 us where they are still in the
// last cache.  One launch that holds x and dy of an image's groups in registers and LDS (512 threads, 25 vectors each)
// needs 48 - 52 us and 5 for the coefficients: it reads less, but its reads, arithmetic and writes follow one another.
// ---- first launch: sums of d and d h over a chunk, by channel and (with the weights) by group -------
template <class XT, class YT, int VEC, bool SILU>
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
    constexpr int B = VEC * XT::ES > 16 || VEC * YT::ES > 16 ? 2 : 4;   // pixels in flight
    for (int q = w.p0 + w.row; q < w.p1; q += B * p.rows) {
      typename DenseVec<XT, VEC>::vec_t rx[B];
      typename DenseVec<YT, VEC>::vec_t rg[B];
#pragma unroll
      for (int u = 0; u < B; ++u) {   // (past the end: the last pixel again, left out of the sums)
        const int at = q + u * p.rows < w.p1 ? q + u * p.rows : w.p1 - 1;
        rx[u] = DenseVec<XT, VEC>::read(x + (int64_t)at * p.pixel);
        rg[u] = DenseVec<YT, VEC>::read(dy + (int64_t)at * p.pixel);
      }
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (q + u * p.rows >= w.p1) break;
        float v[VEC], g[VEC];
        DenseVec<XT, VEC>::widen(rx[u], v);
        DenseVec<YT, VEC>::widen(rg[u], g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float t = v[i] - ch.mean[i];
          const float d = ch.template d<SILU>(i, t, g[i], p.low);
          a1[i] += d;
          a2[i] += d * t;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      s1[(w.row * p.cols + w.col) * VEC + i] = a1[i];
      s2[(w.row * p.cols + w.col) * VEC + i] = a2[i] * ch.rstd[i];
    }
  }
  __syncthreads();
  // ---- the pixel rows meet, in their order: in 64 bits from here to dweight and dbias (a few additions a channel: the error
  // of 2x9x33x35x48 fp32 halves, its time stays at 13.1 us).  A lane's own sums, a few dozen pixels, stay fp32, and so does dx.
  float* const cp = p.cpart + ((int64_t)blockIdx.x * p.C + w.c0) * 2;
  for (int c = threadIdx.x; c < w.width; c += kGnThreads) {
    double a = 0., b = 0.;
    for (int r = 0; r < p.rows; ++r) {
      a += s1[r * p.cols * VEC + c];
      b += s2[r * p.cols * VEC + c];
    }
    cp[c * 2] = (float)a;
    cp[c * 2 + 1] = (float)b;
    const float weight = p.weight ? load_any(p.weight, w.c0 + c, p.affine_dtype) : 1.f;
    s1[c] = (float)a * weight;   // (row 0: read above by this thread only)
    s2[c] = (float)b * weight;
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
  const int rows = p.N * p.chunks;   // (one-launch kernel: a row an image)
  typedef float v2f __attribute__((ext_vector_type(2)));
  double a = 0., b = 0.;
  if (c < p.C) {
    const v2f* const at = (const v2f*)p.cpart + c;
    int r = r0;
    for (; r + 7 * 16 < rows; r += 8 * 16) {   // eight rows in flight
      v2f v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = at[(int64_t)(r + u * 16) * p.C];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        a += v[u][0];
        b += v[u][1];
      }
    }
    for (; r < rows; r += 16) {
      const v2f v = at[(int64_t)r * p.C];
      a += v[0];
      b += v[1];
    }
  }
  s1[t] = (float)a;
  s2[t] = (float)b;
  __syncthreads();
  if (t < 16 && c < p.C) {
    a = b = 0.;
    for (int r = 0; r < 16; ++r) {
      a += s1[r * 16 + t];
      b += s2[r * 16 + t];
    }
    if (p.dbias) p.dbias[c] = (float)a;
    if (p.dweight) p.dweight[c] = (float)b;
  }
}

// ---- second launch: dx; in front of the workgroups of the tiles those of dweight and dbias (`more` of them: their
// sums are the longest chain of the launch) ----------------------------------------------------------------------
template <class XT, class YT, int VEC, bool SILU>
__global__ __launch_bounds__(kGnThreads) void amos_gn_gradient_apply(const GnParams p, int more) {
  __shared__ float s1[kGnThreads * VEC], s2[kGnThreads * VEC];   // by group of the tile: E[d weight], E[d weight h]
  if ((int)blockIdx.x < more) {
    if (blockIdx.y == 0) gn_coefficient_gradients(p, (int)blockIdx.x, s1, s2);
    return;
  }
  const GnTile w = gn_tile<VEC>(p, (int)blockIdx.x - more);
  const GnChannels<VEC> ch(p, w.n, w.c0 + (w.active ? w.col * VEC : 0));
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
  float e1[VEC], e2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int g = fast_div(w.c0 + w.col * VEC + i, p.by_cpg) - w.g0;
    e1[i] = s1[g] * ch.rstd[i];
    e2[i] = s2[g] * ch.rstd[i] * ch.rstd[i];
  }
  const int64_t base = w.n * p.image + w.c0 + w.col * VEC;
  const typename XT::raw_t* const x = (const typename XT::raw_t*)p.x + base;
  const typename YT::raw_t* const dy = (const typename YT::raw_t*)p.dy + base;
  typename XT::raw_t* const dx = (typename XT::raw_t*)p.out + base;
  constexpr int B = VEC * XT::ES > 16 || VEC * YT::ES > 16 ? 2 : 4;   // pixels in flight
  for (int q = w.p0 + w.row; q < w.p1; q += B * p.rows) {
    typename DenseVec<XT, VEC>::vec_t rx[B];
    typename DenseVec<YT, VEC>::vec_t rg[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int at = q + u * p.rows < w.p1 ? q + u * p.rows : w.p1 - 1;
      rx[u] = DenseVec<XT, VEC>::read(x + (int64_t)at * p.pixel);
      rg[u] = DenseVec<YT, VEC>::read(dy + (int64_t)at * p.pixel);
    }
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (q + u * p.rows >= w.p1) break;
      float v[VEC], g[VEC];
      DenseVec<XT, VEC>::widen(rx[u], v);
      DenseVec<YT, VEC>::widen(rg[u], g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float t = v[i] - ch.mean[i];
        v[i] = ch.template d<SILU>(i, t, g[i], p.low) * ch.a[i] - (t * e2[i] + e1[i]);
      }
      DenseVec<XT, VEC>::store(dx + (int64_t)(q + u * p.rows) * p.pixel, v);
    }
  }
}

// Channel totals of a slab from `parts` rows of partial sums in LDS ([part][ct]); dweight, dbias or this image's share of
// them; then the groups' E[d weight] (e1) and E[d weight h] (e2).  A barrier in front of it and behind.
__device__ __forceinline__ void gn_slab_totals(const GnParams& p, const GnSlab& w, int parts, float* s1, float* s2, float* e1, float* e2) {
  const int T = (int)blockDim.x, t = threadIdx.x;
  for (int c = t; c < p.ct; c += T) {
    double a64 = 0., b64 = 0.;
    for (int r = 0; r < parts; ++r) {
      a64 += s1[r * p.ct + c];
      b64 += s2[r * p.ct + c];
    }
    const float a = (float)a64, b = (float)b64;
    const int at = w.c0 + c;
    if (p.N == 1) {
      if (p.dbias) p.dbias[at] = a;
      if (p.dweight) p.dweight[at] = b;
    } else if (p.dbias || p.dweight) {
      float* const cp = p.cpart + ((int64_t)w.n * p.C + at) * 2;
      cp[0] = a;
      cp[1] = b;
    }
    const float weight = p.weight ? load_any(p.weight, at, p.affine_dtype) : 1.f;
    s1[c] = a * weight;
    s2[c] = b * weight;
  }
  __syncthreads();
  {
    int team = 64;
    while (team > 1 && team * w.groups > T) team >>= 1;
    const int lane = t & (team - 1);
    const float count = (float)p.P * p.cpg;
    for (int g = t / team; g < w.groups; g += T / team) {
      float a = 0.f, b = 0.f;
      for (int e = lane; e < p.cpg; e += team) {
        a += s1[g * p.cpg + e];
        b += s2[g * p.cpg + e];
      }
      a = gn_team_sum(a, team);
      b = gn_team_sum(b, team);
      if (lane == 0) {
        e1[g] = a / count;
        e2[g] = b / count;
      }
    }
  }
  __syncthreads();
}

// ---- one launch: x and dy of a slab of whole groups stay in registers between the sums and dx -----------
template <class XT, class YT, int VEC, int R, bool SILU>
__global__ __launch_bounds__(1024) void amos_gn_gradient_held(const GnParams p) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  typedef DenseVec<XT, VEC> VX;
  typedef DenseVec<YT, VEC> VY;
  const GnSlab w = gn_slab(p, VEC);
  const int T = (int)blockDim.x, t = threadIdx.x;
  float *const s1 = lds, *const s2 = lds + p.rows * p.ct, *const e1 = lds + 2 * p.rows * p.ct, *const e2 = e1 + w.groups;
  const int64_t base = w.n * p.image + w.c;
  typename VX::vec_t rx[R];
  typename VY::vec_t rg[R];
  const int c0 = w.active ? w.c : w.c0;
  if (w.active) {
#pragma unroll
    for (int r = 0; r < R; ++r) {   // (pixels past the end: the last one again, left out of the sums)
      const int q = w.row + r * p.rows < p.P ? w.row + r * p.rows : p.P - 1;
      rx[r] = VX::read((const typename XT::raw_t*)p.x + base + (int64_t)q * p.pixel);
      rg[r] = VY::read((const typename YT::raw_t*)p.dy + base + (int64_t)q * p.pixel);
    }
  }
  const GnChannels<VEC> ch(p, w.n, c0);
  if (w.active) {
    float a1[VEC], a2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) a1[i] = a2[i] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (w.row + r * p.rows >= p.P) break;
      float v[VEC], g[VEC];
      VX::widen(rx[r], v);
      VY::widen(rg[r], g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float t = v[i] - ch.mean[i];
        const float d = ch.template d<SILU>(i, t, g[i], p.low);
        a1[i] += d;
        a2[i] += d * t;
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      s1[w.row * p.ct + w.col * VEC + i] = a1[i];
      s2[w.row * p.ct + w.col * VEC + i] = a2[i] * ch.rstd[i];
    }
  }
  __syncthreads();
  // ---- the pixel rows meet: up to `parts` threads a channel, then one
  int parts = T / p.ct < 32 ? T / p.ct : 32;
  if (parts > p.rows) parts = p.rows;
  if (parts > 1) {
    const int c = t % p.ct, part = t / p.ct;
    double a = 0., b = 0.;
    if (part < parts) {
      for (int r = part; r < p.rows; r += parts) {
        a += s1[r * p.ct + c];
        b += s2[r * p.ct + c];
      }
      s1[part * p.ct + c] = (float)a;   // (row `part`: read by this thread only)
      s2[part * p.ct + c] = (float)b;
    }
    __syncthreads();
  } else {
    parts = p.rows;
  }
  gn_slab_totals(p, w, parts, s1, s2, e1, e2);
  if (!w.active) return;
  float m1[VEC], m2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int g = fast_div(w.c + i, p.by_cpg) - w.g0;
    m1[i] = e1[g] * ch.rstd[i];
    m2[i] = e2[g] * ch.rstd[i] * ch.rstd[i];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int q = w.row + r * p.rows;
    if (q >= p.P) break;
    float v[VEC], g[VEC];
    VX::widen(rx[r], v);
    VY::widen(rg[r], g);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float t = v[i] - ch.mean[i];
      v[i] = ch.template d<SILU>(i, t, g[i], p.low) * ch.a[i] - (t * m2[i] + m1[i]);
    }
    VX::store((typename XT::raw_t*)p.out + base + (int64_t)q * p.pixel, v);
  }
}

// dweight and dbias from the images' shares
template <class XT>   // (an instance of its own in every unit)
__global__ __launch_bounds__(kGnThreads) void amos_gn_coefficients(const GnParams p) {
  __shared__ float s1[kGnThreads], s2[kGnThreads];
  gn_coefficient_gradients(p, (int)blockIdx.x, s1, s2);
}

template <class XT, class YT, int VEC, int R, bool SILU>
int launch_gradient_held(const GnParams& p, const GnPlan& plan, hipStream_t stream) {
  void (*const fn)(const GnParams) = amos_gn_gradient_held<XT, YT, VEC, R, SILU>;
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_lds((const void*)fn, 96 * 1024, false, "amos_gn_gradient_held", done)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)((int64_t)p.N * p.tiles)), dim3((unsigned)plan.threads), plan.lds, stream, p);
  if (p.N > 1 && (p.dweight || p.dbias)) hipLaunchKernelGGL((amos_gn_coefficients<XT>), dim3((unsigned)((p.C + 15) / 16)), dim3(kGnThreads), 0, stream, p);
  return 0;
}
template <class XT, class YT, int VEC, bool SILU>
int launch_gradient_tiles(const GnParams& p, hipStream_t stream) {
  const unsigned work = (unsigned)((int64_t)p.N * p.chunks);
  const unsigned more = p.dweight || p.dbias ? (unsigned)((p.C + 15) / 16) : 0;
  hipLaunchKernelGGL((amos_gn_gradient_partial<XT, YT, VEC, SILU>), dim3(work, (unsigned)p.tiles), dim3(kGnThreads), 0, stream, p);
  hipLaunchKernelGGL((amos_gn_gradient_apply<XT, YT, VEC, SILU>), dim3(work + more, (unsigned)p.tiles), dim3(kGnThreads), 0, stream, p, (int)more);
  return 0;
}
template <class XT, class YT, bool SILU>
int launch_gradient_kernels(const GnParams& p, const GnPlan& plan, hipStream_t stream) {
  constexpr int WIDE = XT::ES == 4 || YT::ES == 4 ? 4 : 8;   // 16 bytes of the wider type
  if (!plan.held) return plan.vec == WIDE ? launch_gradient_tiles<XT, YT, WIDE, SILU>(p, stream) : launch_gradient_tiles<XT, YT, 1, SILU>(p, stream);
  if (plan.vec == WIDE)
    return plan.held <= 2 ? launch_gradient_held<XT, YT, WIDE, 2, SILU>(p, plan, stream) : launch_gradient_held<XT, YT, WIDE, kGnHeldGradient, SILU>(p, plan, stream);
  return plan.held <= 2 ? launch_gradient_held<XT, YT, 1, 2, SILU>(p, plan, stream) : launch_gradient_held<XT, YT, 1, kGnHeldGradient, SILU>(p, plan, stream);
}
template <class XT, class YT>
int launch_gradient_act(const GnParams& p, const GnPlan& plan, hipStream_t stream) {
  return p.act == AMOS_ACT_SILU ? launch_gradient_kernels<XT, YT, true>(p, plan, stream) : launch_gradient_kernels<XT, YT, false>(p, plan, stream);
}
template <class XT>
int launch_gradient(const GnParams& p, const GnPlan& plan, hipStream_t stream) {
  if (p.y_dtype == AMOS_F32) return launch_gradient_act<XT, TypeF32>(p, plan, stream);
  if (p.y_dtype == AMOS_F16) return launch_gradient_act<XT, TypeF16>(p, plan, stream);
  return launch_gradient_act<XT, TypeBF16>(p, plan, stream);
}

}  // namespace amos
