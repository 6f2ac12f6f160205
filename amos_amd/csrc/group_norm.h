// Group norm with an activation over channels-last tensors, and its gradient, for gfx950.
//
//   per image n and group g of C / groups channels, over its pixels and channels:
//     mean, var = E[x], E[(x - mean)^2];  h = (x - mean) / sqrt(var + eps)
//     z = h weight[c] + bias[c];  y = act(z),  act none, relu or silu (z / (1 + exp(-z)))
//   gradient, with d = dy act'(z):
//     dweight[c] = sum d h,  dbias[c] = sum d      (over images and pixels)
//     dx = (d weight - E[d weight] - h E[d weight h]) / sqrt(var + eps)   (E over the group)
//
// Both move bytes.  Where whole groups of an image fit into a workgroup's registers, one launch reads
// the tensors once and writes ("held"); else a launch reads them for the sums and a second one
// reads them again and writes.  There a workgroup takes a run of pixels ("chunk") and a tile of channels; a
// lane keeps VEC neighbouring channels and strides over pixels, so that a wave's loads are whole rows.  Sums are
// joined in a fixed order (no atomics: the same bits on every run).
// 16 x 128 x 128 x 256 bf16 + silu in two launches: forward 87 us, 4.6 TB/s over its three passes (a large copy: 5.1),
// gradient 144 us, 4.7 TB/s over five; 1 x 128 x 128 x 512: 18 and 23 us (with tiles of all channels, 128 workgroups: 36
// and 41).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dense_type.h"
#include "fast_div.h"

namespace amos {

constexpr int kGnThreads = 256;

struct GnParams {
  const void* x;
  const void* dy;            // gradient only
  void* out;                 // y, dx
  const void* weight;        // [C] or null (ones), of type affine_dtype
  const void* bias;          // [C] or null (zeros)
  float* mean;               // [N][G]: written by the forward launch, read by the gradient
  float* rstd;
  float* dweight;            // [C] or null
  float* dbias;
  float* part;               // workspace: see GnPlan
  float* cpart;
  int64_t image, pixel;      // elements between images, between pixels
  int N, P, C, G, cpg;       // pixels of an image, channels, groups, channels of a group
  int ct, tiles, sub;        // channels of a tile, tiles, tiles of a group (1 where a tile holds whole groups)
  int cols, rows;            // threads across a tile's channels, pixels side by side
  int chunk, chunks;         // pixels of a chunk, chunks of an image
  int slots;                 // partial results of a group: chunks * sub
  float eps;
  int act, affine_dtype;
  float low;                 // act none: NaN, relu: 0 (what z is not let below)
  FastDiv by_cpg, by_cols;
  FastDiv by_epg;            // one-launch kernels: entries of a group in a row of threads
  int y_dtype;
};

// 1 / sqrt(var + eps).  Sums are fp32: a variance that left their range (deviations from some 2^64 / sqrt(elements of the
// group) up) is no variance, and its group's results are NaN, not the bias that a factor of 1 / infinity would leave
__device__ __forceinline__ float gn_rstd(float var, float eps) {
  const float v = var + eps;
  return v < __builtin_inff() ? 1.f / sqrtf(v) : __builtin_nanf("");
}

// 1 / (1 + exp(-z)), from z times -log2(e).  Exponential and reciprocal are single instructions, each right to its last
// place, and the factor's rounding makes silu off by some (|z| + 4) 2^-23 of itself; with exp2f and a division
// 32 x 56 x 56 x 256 bf16 takes 40.6 us instead of 32.2 (inputs from memory), its gradient 63.9 instead of 57.7.
__device__ __forceinline__ float gn_sigmoid2(float scaled) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(scaled)); }
constexpr float kGnLog2e = 1.44269504088896341f;
// The activations without a branch an element: silu is a kernel's own instance; none and relu are z no lower than
// `low`, NaN or 0 (comparisons that are false for NaN: a z of NaN stays, and without an activation every z passes)
template <bool SILU>
__device__ __forceinline__ float gn_act(float z, float low) {
  if constexpr (SILU) return z * gn_sigmoid2(z * -kGnLog2e);
  else return z < low ? low : z;
}
template <bool SILU>
__device__ __forceinline__ float gn_act_gradient(float dy, float z, float low) {   // dy act'(z)
  if constexpr (SILU) {
    const float s = gn_sigmoid2(z * -kGnLog2e);
    return dy * (s * (1.f + z * (1.f - s)));
  } else {
    return z <= low ? 0.f : dy;
  }
}

// where a workgroup works
struct GnTile {
  int n, chunk, tile, c0, width;   // image, chunk, tile, first channel and channels of the tile
  int g0, groups;                  // first group, groups the tile meets
  int p0, p1;                      // pixels
  int col, row;                    // of this thread
  bool active;
};
template <int VEC>
__device__ __forceinline__ GnTile gn_tile(const GnParams& p, int block) {
  GnTile w;
  w.tile = blockIdx.y;
  w.n = block / p.chunks;
  w.chunk = block - w.n * p.chunks;
  w.c0 = w.tile * p.ct;
  if (p.sub > 1) {   // tiles inside a group: the last of a group may be narrower
    w.g0 = w.tile / p.sub;
    const int s = w.tile - w.g0 * p.sub;
    w.c0 = w.g0 * p.cpg + s * p.ct;
    w.width = p.cpg - s * p.ct < p.ct ? p.cpg - s * p.ct : p.ct;
    w.groups = 1;
  } else {
    w.g0 = w.c0 / p.cpg;
    w.width = p.C - w.c0 < p.ct ? p.C - w.c0 : p.ct;
    w.groups = w.width / p.cpg;
  }
  w.p0 = w.chunk * p.chunk;
  w.p1 = w.p0 + p.chunk < p.P ? w.p0 + p.chunk : p.P;
  const int t = threadIdx.x;
  w.row = fast_div(t, p.by_cols);
  w.col = t - w.row * p.cols;
  w.active = w.row < p.rows && w.col * VEC < w.width;
  return w;
}

// threads that share a group of a tile: a power of two inside a wave
__device__ __forceinline__ int gn_team(int groups) {
  int team = 64;
  while (team > 1 && team * groups > kGnThreads) team >>= 1;
  return team;
}
__device__ __forceinline__ float gn_team_sum(float v, int team) {
  for (int s = 1; s < team; s <<= 1) v += __shfl_xor(v, s, 64);
  return v;
}

struct GnPlan {
  int vec;
  bool uni;                  // a vector lies inside one group
  int held;                  // pixels a thread of the one-launch kernel holds (0: two launches)
  int threads, lds;          // of that kernel
  int64_t part_floats, cpart_floats;
};

// ---- the one-launch kernels: a slab of whole groups of one image is held in registers -------------
// A workgroup takes p.ct channels (whole groups) of one image; a lane keeps VEC channels of the pixels row,
// row + rows, ...  UNI: a vector lies inside one group.
struct GnSlab {
  int n, c0, g0, groups;
  int col, row, c;               // of this thread; its first channel
  bool active;
};
__device__ __forceinline__ GnSlab gn_slab(const GnParams& p, int vec) {
  GnSlab w;
  int b = blockIdx.x, slab;
  // slabs of an image share memory lines: where images come in eights, an image's slabs go to one XCD
  // (workgroups are dealt to the eight in launch order)
  if ((p.N & 7) == 0) {
    const int s = b >> 3, image = s / p.tiles;
    w.n = (b & 7) + 8 * image;
    slab = s - image * p.tiles;
  } else {
    w.n = b / p.tiles;
    slab = b - w.n * p.tiles;
  }
  w.c0 = slab * p.ct;
  w.g0 = w.c0 / p.cpg;
  w.groups = p.ct / p.cpg;
  const int t = threadIdx.x;
  w.row = fast_div(t, p.by_cols);
  w.col = t - w.row * p.cols;
  w.active = w.row < p.rows;
  w.c = w.c0 + w.col * vec;
  return w;
}
// Sums over each group of a slab: the threads' values `v` (one each for UNI, else one for each channel) meet in
// `lds` ([rows][entries]), a team of lanes adds a group's, in an order that does not depend on timing; `of` each
// sum in `total` [groups].  Barriers between and behind.
template <int VEC, bool UNI, class F>
__device__ __forceinline__ void gn_group_sums(const GnParams& p, const GnSlab& w, const float* v, float* lds, float* total, F of) {
  const int per = UNI ? p.cols : p.cols * VEC;
  const int epg = per / w.groups;
  if (w.active) {
    if (UNI) lds[w.row * per + w.col] = v[0];
    else
#pragma unroll
      for (int i = 0; i < VEC; ++i) lds[w.row * per + w.col * VEC + i] = v[i];
  }
  __syncthreads();
  int team = 64;
  while (team > 1 && team * w.groups > (int)blockDim.x) team >>= 1;
  const int lane = threadIdx.x & (team - 1), step = (int)blockDim.x / team, entries = p.rows * epg;
  for (int g = threadIdx.x / team; g < w.groups; g += step) {
    float s = 0.f;
    for (int e = lane; e < entries; e += 4 * team) {   // four reads in flight
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = e + u * team, r = fast_div(at, p.by_epg);
        x[u] = at < entries ? lds[r * per + g * epg + (at - r * epg)] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) s += x[u];
    }
    s = gn_team_sum(s, team);
    if (lane == 0) total[g] = of(s);
  }
  __syncthreads();
}

}  // namespace amos
