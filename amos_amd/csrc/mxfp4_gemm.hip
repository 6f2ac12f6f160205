#include "mxfp4_gemm.h"

#include <string.h>

#include <mutex>

#include "mapper.h"
#include "mxfp4_tile_kernel.h"

namespace amos {

// ---- few rows of A ------------------------------------------------------------------------------
// With few tokens the weights B are read once and hardly reused: the call lasts as long as their
// bytes take.  The weights are the matrix instruction's row operand and come from HBM straight into
// registers (no LDS: nothing is shared), tokens are its columns.  A workgroup of eight waves owns
// 16 RT rows of B and up to 16 TT tokens; the waves take K in turns of 512 elements (four
// instructions' worth: 256 contiguous bytes of every row and four words of scales, all loads of a
// turn in flight together) and their sums meet in LDS, added in the order of the waves.
// SRC: what A is -- codes, or (fp32 / fp16 / bf16) elements that are quantised here: a lane's fragment
// is exactly one block, so it finds the block's scale without any exchange.
enum { SRC_MX = 0, SRC_F32 = 1, SRC_F16 = 2, SRC_BF16 = 3 };
template <int SRC> struct SrcType { typedef TypeF32 type; };
template <> struct SrcType<SRC_F16> { typedef TypeF16 type; };
template <> struct SrcType<SRC_BF16> { typedef TypeBF16 type; };

// the block (step, lane group) of token row `m`, quantised
template <class T>
__device__ __forceinline__ void mx_quantize_fragment(const MxGemmParams& p, int64_t m, int64_t k, mx_v4i& codes, int& scale) {
  const typename T::raw_t* const x = (const typename T::raw_t*)p.dense + m * p.K + k;
  float v[32];
  if (p.dense_vec && k + 32 <= p.K) {
    constexpr int N = 16 / T::ES;
#pragma unroll
    for (int i = 0; i < 32; i += N) DenseVec<T, N>::load(x + i, v + i);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = k + i < p.K ? T::widen(x[i]) : 0.f;
  }
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const unsigned b = mx_abs_bits(v[i]);
    top = b > top ? b : top;
  }
  const unsigned s = mx_scale_byte(top);
  scale = (int)s;
#pragma unroll
  for (int i = 0; i < 4; ++i) codes[i] = (int)mx_encode8(v + 8 * i, s);
}

constexpr int kFewWaves = 8, kFewTurn = 4;

template <int SRC, int RT, int TT>
__global__ __launch_bounds__(64 * kFewWaves) void amos_mx_gemm_few(const MxGemmParams p) {
  __shared__ __attribute__((aligned(16))) float sums[kFewWaves][RT * TT][64][4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * (16 * RT), m0 = blockIdx.y * (16 * TT);
  const int64_t pitch = (int64_t)p.steps * 64, spitch = (int64_t)p.steps * 4;
  const unsigned char *brow[RT], *bsc[RT], *arow[TT], *asc[TT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {   // (rows past the end repeat the last one: their sums are not stored)
    const int64_t n = n0 + 16 * i + r < p.N ? n0 + 16 * i + r : p.N - 1;
    brow[i] = p.b + n * pitch + q * 16;
    bsc[i] = p.bs + n * spitch + q;
  }
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    const int64_t m = m0 + 16 * j + r < p.M ? m0 + 16 * j + r : p.M - 1;
    arow[j] = p.a + m * pitch + q * 16;
    asc[j] = p.as + m * spitch + q;
  }
  v4f acc[RT][TT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int s0 = wave * kFewTurn; s0 < p.steps; s0 += kFewWaves * kFewTurn) {
    mx_v4i bf[kFewTurn][RT];
    int bx[kFewTurn][RT];
#pragma unroll
    for (int u = 0; u < kFewTurn; ++u) {
      const int s = s0 + u < p.steps ? s0 + u : p.steps - 1;   // (past the end: loaded again, not multiplied)
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        bf[u][i] = *(const mx_v4i*)(brow[i] + s * 64);
        bx[u][i] = bsc[i][s * 4];
      }
    }
#pragma unroll
    for (int u = 0; u < kFewTurn; ++u) {
      const int s = s0 + u;
      if (s >= p.steps) break;
      mx_v4i af[TT];
      int ax[TT];
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        if constexpr (SRC == SRC_MX) {
          af[j] = *(const mx_v4i*)(arow[j] + s * 64);
          ax[j] = asc[j][s * 4];
        } else {
          const int64_t m = m0 + 16 * j + r;
          af[j] = mx_v4i{0, 0, 0, 0};
          ax[j] = 0;
          if (m < p.M) mx_quantize_fragment<typename SrcType<SRC>::type>(p, m, (int64_t)s * 128 + q * 32, af[j], ax[j]);
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = mx_mfma(bf[u][i], af[j], acc[i][j], bx[u][i], ax[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) *(v4f*)sums[wave][i * TT + j][lane] = acc[i][j];
  __syncthreads();
  for (int slot = t; slot < RT * TT * 64; slot += 64 * kFewWaves) {
    const int tile = slot >> 6, l = slot & 63;
    v4f v = *(const v4f*)sums[0][tile][l];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) {
      const v4f x = *(const v4f*)sums[w][tile][l];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
    const int64_t m = m0 + 16 * (tile % TT) + (l & 15);
    const int n = n0 + 16 * (tile / TT) + 4 * (l >> 4);
    if (m < p.M) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) store_any(p.c, m * p.N + n + e, p.out_dtype, mx_tail(p.tail, v[e], m, n + e, p.N));
    }
  }
}

template <int RT, int TT>
static void launch_few(const MxGemmParams& p, int src, hipStream_t stream) {
  const dim3 grid((unsigned)((p.N + 16 * RT - 1) / (16 * RT)), (unsigned)((p.M + 16 * TT - 1) / (16 * TT))), block(64 * kFewWaves);
  if (src == SRC_MX) hipLaunchKernelGGL((amos_mx_gemm_few<SRC_MX, RT, TT>), grid, block, 0, stream, p);
  else if (src == SRC_F32) hipLaunchKernelGGL((amos_mx_gemm_few<SRC_F32, RT, TT>), grid, block, 0, stream, p);
  else if (src == SRC_F16) hipLaunchKernelGGL((amos_mx_gemm_few<SRC_F16, RT, TT>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((amos_mx_gemm_few<SRC_BF16, RT, TT>), grid, block, 0, stream, p);
}

// ---- many rows of A -----------------------------------------------------------------------------
template <int WI, int WJ, int BI, int BJ>
static int launch_tile(const MxGemmParams& p, hipStream_t stream) {
  constexpr int lds = 2 * (BI + BJ) * 136;
  void (*const fn)(const MxTileParams) = amos_mx_gemm_tile<WI, WJ, BI, BJ>;
  static std::once_flag once;
  static hipError_t err = hipSuccess;
  static int spilled = 0;
  std::call_once(once, [&] {
    err = hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    // (the kernel counts its outstanding copies; register spills would count among them)
    hipFuncAttributes fa;
    if (err == hipSuccess) err = hipFuncGetAttributes(&fa, (const void*)fn);
    if (err == hipSuccess) spilled = (int)fa.localSizeBytes;
  });
  if (err != hipSuccess) return set_error(AMOS_ERR_HIP, "amos_mx_gemm_tile<%dx%d>: %s", BI, BJ, hipGetErrorString(err));
  if (spilled) return set_error(AMOS_ERR_INFEASIBLE, "amos_mx_gemm_tile<%dx%d> was built with scratch memory", BI, BJ);
  MxTileParams t;
  t.g = p;
  t.tiles_i = (p.M + BI - 1) / BI;
  t.tiles_j = (p.N + BJ - 1) / BJ;
  t.per_split = (p.steps + 1) / 2;
  t.slices = nullptr;
  const int es = dense_size(p.out_dtype);
  t.vec_out = ((uintptr_t)p.c & 15) == 0 && ((int64_t)p.N * es) % 16 == 0;
  t.vec_add = p.tail.add && ((uintptr_t)p.tail.add & 15) == 0;   // (N is a multiple of the run then)
  if ((int64_t)t.tiles_i * t.tiles_j >= (int64_t)1 << 31) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product of %d x %d results", p.M, p.N);
  hipLaunchKernelGGL(fn, dim3((unsigned)(t.tiles_i * t.tiles_j), 1), dim3(64 * WI * WJ), lds, stream, t);
  return 0;
}

int mx_quantize(const amos_mxfp4_desc_t* d, const void* x, void* codes, void* scales, hipStream_t stream);

static int check_desc(const amos_mxfp4_gemm_desc_t* d) {
  if (!d) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  if (d->M < 1 || d->N < 1 || d->K < 1)
    return set_error(AMOS_ERR_BAD_ARG, "4-bit product of extents M %lld, N %lld, K %lld", (long long)d->M, (long long)d->N, (long long)d->K);
  const int64_t lim = (int64_t)1 << 31;
  if (d->M >= lim || d->N >= lim || d->K >= lim) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: extents of 2^31 and more");
  if (d->a_dtype != AMOS_MXFP4 && !is_dense_dtype(d->a_dtype))
    return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: A of dtype %d (4 bits, fp32, fp16 or bf16)", d->a_dtype);
  if (!is_dense_dtype(d->out_dtype)) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: output dtype %d (fp32, fp16 or bf16)", d->out_dtype);
  return 0;
}

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// A's rows are quantised by a launch of their own: codes and scales in the workspace
static bool quantize_first(const amos_mxfp4_gemm_desc_t* d) { return d->a_dtype != AMOS_MXFP4; }

static int run(const amos_mxfp4_gemm_desc_t* d, const amos_mxfp4_epilogue_t* e, const void* A, const void* a_scales, const void* B,
               const void* b_scales, void* C, void* workspace, size_t ws_bytes, hipStream_t stream) {
  int rc = check_desc(d);
  if (rc) return rc;
  const bool dense = d->a_dtype != AMOS_MXFP4;
  if (!A || !B || !b_scales || !C || (!dense && !a_scales)) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  if ((((uintptr_t)B | (dense ? 0 : (uintptr_t)A)) & 15) || (((uintptr_t)b_scales | (dense ? 0 : (uintptr_t)a_scales)) & 3))
    return set_error(AMOS_ERR_BAD_ARG, "4-bit product: codes must be 16-byte aligned, scales 4-byte aligned");
  if ((dense && ((uintptr_t)A & (dense_size(d->a_dtype) - 1))) || ((uintptr_t)C & (dense_size(d->out_dtype) - 1)))
    return set_error(AMOS_ERR_BAD_ARG, "4-bit product: misaligned matrix");
  MxGemmParams p;
  memset(&p, 0, sizeof(p));
  if (e) {
    if (e->bias && !is_dense_dtype(e->bias_dtype)) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: bias of dtype %d", e->bias_dtype);
    if (e->add && !is_dense_dtype(e->add_dtype)) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: added operand of dtype %d", e->add_dtype);
    if ((e->bias && ((uintptr_t)e->bias & (dense_size(e->bias_dtype) - 1))) || (e->add && ((uintptr_t)e->add & (dense_size(e->add_dtype) - 1))))
      return set_error(AMOS_ERR_BAD_ARG, "4-bit product: misaligned bias or added operand");
    p.tail.bias = e->bias;
    p.tail.add = e->add;
    p.tail.bias_dtype = e->bias_dtype;
    p.tail.add_dtype = e->add_dtype;
  }
  p.b = (const unsigned char*)B;
  p.bs = (const unsigned char*)b_scales;
  p.c = C;
  p.M = (int)d->M;
  p.N = (int)d->N;
  p.K = (int)d->K;
  p.steps = (int)(mx_pitch(d->K) / 64);
  p.out_dtype = d->out_dtype;
  int src = SRC_MX;
  if (quantize_first(d)) {
    const int64_t code_bytes = round256(d->M * mx_pitch(d->K));
    if (!workspace || ws_bytes < amos_mxfp4_gemm_workspace_bytes(d) || ((uintptr_t)workspace & 255))
      return set_error(AMOS_ERR_WORKSPACE, "4-bit product: %zu bytes of 256-byte aligned workspace wanted for A's codes", amos_mxfp4_gemm_workspace_bytes(d));
    unsigned char* const codes = (unsigned char*)workspace;
    amos_mxfp4_desc_t q;
    memset(&q, 0, sizeof(q));
    q.rows = d->M;
    q.cols = d->K;
    q.dtype = d->a_dtype;
    q.axis = 1;
    rc = mx_quantize(&q, A, codes, codes + code_bytes, stream);
    if (rc) return rc;
    p.a = codes;
    p.as = codes + code_bytes;
  } else {
    p.a = (const unsigned char*)A;
    p.as = (const unsigned char*)a_scales;
  }
  // (the tiled kernel's offsets inside a tile have 32 bits)
  if (d->M > 64 && p.steps < 1 << 18) {
    const int64_t big = ((d->M + 255) / 256) * ((d->N + 255) / 256);
    rc = big >= 256 ? launch_tile<4, 2, 256, 256>(p, stream) : launch_tile<2, 4, 128, 128>(p, stream);
    if (rc) return rc;
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(err));
    return 0;
  }
  if ((d->M + 63) / 64 > 65535) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product of more than %d rows", 65535 * 64);
  if (d->M <= 16) launch_few<1, 1>(p, src, stream);
  else if (d->M <= 32) launch_few<2, 2>(p, src, stream);
  else launch_few<2, 4>(p, src, stream);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(err));
  return 0;
}

}  // namespace amos

using namespace amos;

extern "C" {

size_t amos_mxfp4_gemm_workspace_bytes(const amos_mxfp4_gemm_desc_t* desc) {
  if (check_desc(desc)) return 0;
  if (!quantize_first(desc)) return 0;
  const int64_t pitch = mx_pitch(desc->K);
  return (size_t)(round256(desc->M * pitch) + round256(desc->M * (pitch / 16)));
}

int amos_mxfp4_gemm(const amos_mxfp4_gemm_desc_t* desc, const amos_mxfp4_epilogue_t* epilogue, const void* A, const void* a_scales,
                    const void* B, const void* b_scales, void* C, void* workspace, size_t ws_bytes, void* stream) {
  return run(desc, epilogue, A, a_scales, B, b_scales, C, workspace, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
