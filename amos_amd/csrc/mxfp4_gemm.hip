#include "mxfp4_gemm.h"

#include <string.h>

#include "lds_limit.h"
#include "mapper.h"
#include "mxfp4_tile_kernel.h"

namespace amos {

// ---- few rows of A ------------------------------------------------------------------------------
// With few tokens the weights B are read once and hardly reused: the call lasts as long as their
// bytes take.  The weights are the matrix instruction's row operand and come from memory straight into
// registers (no LDS: nothing is shared), tokens are its columns.  A workgroup owns 16 RT rows of B and up
// to 16 TT tokens; its waves take K in turns of 512 elements (four instructions' worth: 256 contiguous
// bytes of every row), and there are as many waves, up to 16, as give each one turn: all of a wave's loads
// are in flight together.  A row's scales of a turn are one 16-byte load.  The waves' sums meet in LDS,
// added in the order of the waves.  1 x 4096 x 4096 (8.9 MB of weights) 5.4 us, 1 x 16384 x 4096 (36 MB) 9.0 us = 4.0 TB/s;
// a launch that does nothing takes some 2.5 us of that.
// SRC: what A is -- codes, or (fp32 / fp16 / bf16) elements that are quantised here: a lane's fragment
// is exactly one block, so it finds the block's scale without any exchange.
enum { SRC_MX = 0, SRC_F32 = 1, SRC_F16 = 2, SRC_BF16 = 3 };
template <int SRC> struct SrcType { typedef TypeF32 type; };
template <> struct SrcType<SRC_F16> { typedef TypeF16 type; };
template <> struct SrcType<SRC_BF16> { typedef TypeBF16 type; };

// the block of token row `m` that starts at element k, quantised
template <class T>
__device__ __forceinline__ void mx_quantize_fragment(const MxGemmParams& p, int64_t m, int64_t k, mx_v4i& codes, int& scale) {
  const typename T::raw_t* const x = (const typename T::raw_t*)p.dense + m * p.K + k;
  float v[32];
  if (k + 32 <= p.K) {
    constexpr int N = 16 / T::ES;
    typename DenseVec<T, N>::vec_t raw[32 / N];
#pragma unroll
    for (int i = 0; i < 32 / N; ++i) raw[i] = DenseVec<T, N>::read(x + i * N);
#pragma unroll
    for (int i = 0; i < 32 / N; ++i) DenseVec<T, N>::widen(raw[i], v + i * N);
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

constexpr int kTurn = 4;
typedef int mx_v4i_words __attribute__((ext_vector_type(4), aligned(4)));

// a turn of one row's fragments and scales.  `here` (uniform) of its kTurn steps exist; past them: the last step again
__device__ __forceinline__ void mx_load_turn(const unsigned char* codes, const unsigned char* scales, int s0, int here, int q, mx_v4i* f, mx_v4i& x) {
#pragma unroll
  for (int u = 0; u < kTurn; ++u) f[u] = *(const mx_v4i*)(codes + (int64_t)(s0 + (u < here ? u : here - 1)) * 64 + q * 16);
  if (here == kTurn) {
    x = *(const mx_v4i_words*)(scales + (int64_t)s0 * 4);
  } else {
#pragma unroll
    for (int u = 0; u < kTurn; ++u) x[u] = *(const int*)(scales + (int64_t)(s0 + (u < here ? u : here - 1)) * 4);
  }
}

template <int SRC, int RT, int TT, int MAXW>
__global__ __launch_bounds__(64 * MAXW) void amos_mx_gemm_few(const MxGemmParams p) {
  extern __shared__ __attribute__((aligned(16))) float sums[];   // [waves][RT * TT][64][4]
  const int t = threadIdx.x, lane = t & 63, waves = (int)blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * (16 * RT), m0 = blockIdx.y * (16 * TT);
  const int64_t pitch = (int64_t)p.steps * 64, spitch = (int64_t)p.steps * 4;
  v4f acc[RT][TT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int s0 = wave * kTurn; s0 < p.steps; s0 += waves * kTurn) {
    const int here = p.steps - s0 < kTurn ? p.steps - s0 : kTurn;
    mx_v4i bf[RT][kTurn], bx[RT];
    mx_v4i af[TT][kTurn], ax[TT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {   // (rows past the end repeat the last one: their sums are not stored)
      const int64_t n = n0 + 16 * i + r < p.N ? n0 + 16 * i + r : p.N - 1;
      mx_load_turn(p.b + n * pitch, p.bs + n * spitch, s0, here, q, bf[i], bx[i]);
    }
    if constexpr (SRC == SRC_MX) {
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        const int64_t m = m0 + 16 * j + r < p.M ? m0 + 16 * j + r : p.M - 1;
        mx_load_turn(p.a + m * pitch, p.as + m * spitch, s0, here, q, af[j], ax[j]);
      }
    }
#pragma unroll
    for (int u = 0; u < kTurn; ++u) {
      if (u >= here) break;
      int xa[TT];
      if constexpr (SRC == SRC_MX) {
#pragma unroll
        for (int j = 0; j < TT; ++j) xa[j] = (int)((unsigned)ax[j][u] >> (8 * q));   // (the instruction takes the lowest byte)
      } else {
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          const int64_t m = m0 + 16 * j + r;
          af[j][u] = mx_v4i{0, 0, 0, 0};
          xa[j] = 0;
          if (m < p.M) mx_quantize_fragment<typename SrcType<SRC>::type>(p, m, (int64_t)(s0 + u) * 128 + q * 32, af[j][u], xa[j]);
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int xb = (int)((unsigned)bx[i][u] >> (8 * q));
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = mx_mfma(bf[i][u], af[j][u], acc[i][j], xb, xa[j]);
      }
    }
  }
  if (waves > 1) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j) *(v4f*)(sums + (((wave * RT + i) * TT + j) * 64 + lane) * 4) = acc[i][j];
    __syncthreads();
  }
  // a lane's four sums: rows 4q .. 4q + 3 of B for one token, neighbours in C
  auto finish = [&](int i, int j, int l, v4f v) {
    const int64_t m = m0 + 16 * j + (l & 15);
    const int n = n0 + 16 * i + 4 * (l >> 4);
    if (m >= p.M || n >= p.N) return;
    const int64_t at = m * p.N + n;
    if (n + 4 <= p.N) {
      float e[4];
      if (p.tail.bias) {
        load_run_any<4>(p.tail.bias, n, p.tail.bias_dtype, 0.f, e);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += e[k];
      }
      if (p.tail.add) {
        load_run_any<4>(p.tail.add, at, p.tail.add_dtype, 0.f, e);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += e[k];
      }
      const float w[4] = {v[0], v[1], v[2], v[3]};
      store_run_any<4>(p.c, at, p.out_dtype, w);
    } else {
      for (int k = 0; k < 4 && n + k < p.N; ++k) store_any(p.c, at + k, p.out_dtype, mx_tail(p.tail, v[k], m, n + k, p.N));
    }
  };
  if (waves == 1) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j) finish(i, j, lane, acc[i][j]);
    return;
  }
  for (int slot = t; slot < RT * TT * 64; slot += (int)blockDim.x) {
    const int tile = slot >> 6, l = slot & 63;
    v4f v = *(const v4f*)(sums + (tile * 64 + l) * 4);
    for (int w = 1; w < waves; ++w) {
      const v4f x = *(const v4f*)(sums + ((w * RT * TT + tile) * 64 + l) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
    finish(tile / TT, tile % TT, l, v);
  }
}

constexpr int64_t kGridThreads = (int64_t)1 << 32;   // a grid's first extent has fewer
template <int SRC, int RT, int TT>
static int launch_few(const MxGemmParams& p, hipStream_t stream) {
  constexpr int MAXW = TT == 1 ? 16 : 8;   // (the waves' sums: at most 64 KB)
  int waves = (p.steps + kTurn - 1) / kTurn;
  if (waves > MAXW) waves = MAXW;
  const int64_t gy = ((int64_t)p.M + 16 * TT - 1) / (16 * TT);
  const int64_t gx = ((int64_t)p.N + 16 * RT - 1) / (16 * RT);
  if (gy > 65535 || gx * 64 * waves >= kGridThreads) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product of %d x %d results and K %d", p.M, p.N, p.K);
  const size_t lds = waves > 1 ? (size_t)waves * RT * TT * 1024 : 0;
  hipLaunchKernelGGL((amos_mx_gemm_few<SRC, RT, TT, MAXW>), dim3((unsigned)gx, (unsigned)gy),
                     dim3((unsigned)(64 * waves)), lds, stream, p);
  return 0;
}

// Row blocks a workgroup takes.  Every workgroup reads all of its tokens' codes, and what limits it then is the rate of
// its load instructions; so a grid that one round of the 256 compute units can take is given as few workgroups as
// that (24 x 4096 x 4096: 1, 2 blocks 5.7, 7.1 us; 32 x 8192 x 2048: 5.8, 4.9 us; 8 x 10240 x 8192: 1, 2, 3 blocks 14.9, 15.7, 11.7 us),
// longer ones one block a workgroup (1 x 16384 x 4096: 1, 2, 3 blocks 9.0, 9.0, 11.1 us).
static int few_blocks(int64_t blocks) {
  const int64_t rt = (blocks + 255) / 256;
  return rt <= 3 ? (int)rt : 1;
}

// ---- many rows of A -----------------------------------------------------------------------------
template <int WI, int WJ, int BI, int BJ, int NS, bool FLAT>
static int launch_tile(const MxGemmParams& p, hipStream_t stream) {
  constexpr int lds = (BI + BJ) * (NS * 128 + 64);
  void (*const fn)(const MxTileParams) = amos_mx_gemm_tile<WI, WJ, BI, BJ, NS, FLAT>;
  MxTileParams t;
  t.g = p;
  t.tiles_i = (p.M + BI - 1) / BI;
  t.tiles_j = (p.N + BJ - 1) / BJ;
  t.stream_out = (int64_t)p.M * p.N * 4 > (int64_t)32 << 20;
  t.vec_scales = p.steps >= 4;
  if ((int64_t)t.tiles_i * t.tiles_j * 64 * WI * WJ >= kGridThreads) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product of %d x %d results", p.M, p.N);
  static std::atomic<uint64_t> done{0};
  if (const int rc = allow_lds((const void*)fn, lds, true, "amos_mx_gemm_tile", done)) return rc;
  hipLaunchKernelGGL(fn, dim3((unsigned)(t.tiles_i * t.tiles_j)), dim3(64 * WI * WJ), lds, stream, t);
  return 0;
}

// The tile: the one whose rounds of the 256 compute units take the least time.  `one`, `two`: microseconds of a round with
// one and with two workgroups a unit (the larger tiles' LDS leaves room for one), all at K = 4096; at other K the ratios
// hold well enough (every tile timed on 48 drawn shapes of 34 to 8232 rows, 77 to 10770 columns, K 257 to 7541: the one
// chosen is at most 7 % behind the best of the five, 0.6 % on the mean).
//   2048 x 2048 x 2048: 128x128 10.6 us, 64x64 14.5, 256x256 19.6      4096 x 2048 x 4096: 128x256 24.1 us, 128x128 28.5, 256x256 33.6
//   333 x 1000 x 2050: 32x64 5.4 us, 64x64 6.1                         3000 x 3000 x 1000: 256x256 15.0 us, 128x256 18.4, 128x128 19.4
// Four stages and a step's fragments read at once let 128x128 in one round wait for neither memory nor LDS (1024 x 4096 x 4096:
// 15.7 us; three stages with phases 20.3, two workgroups a unit with two stages 19.9).
struct TileCost {
  int bi, bj;
  double one, two;
};
constexpr TileCost kTiles[] = {{32, 64, 7.0, 9.4}, {64, 64, 8.6, 12.3}, {128, 128, 16.0, 32.0}, {128, 256, 24.1, 48.2}, {256, 256, 38.5, 77.0}};
static int pick_tile(int64_t M, int64_t N) {   // -> index
  int best = 0;
  double least = 0;
  for (int i = 0; i < 5; ++i) {
    const TileCost& t = kTiles[i];
    const int64_t n = ((M + t.bi - 1) / t.bi) * ((N + t.bj - 1) / t.bj), rest = n % 512;
    const double cost = (double)(n / 512) * t.two + (rest > 256 ? t.two : rest ? t.one : 0.0);
    if (i == 0 || cost < least) {
      best = i;
      least = cost;
    }
  }
  return M <= 32 ? 0 : best;
}

int mx_quantize(const amos_mxfp4_desc_t* d, const void* x, void* codes, void* scales, hipStream_t stream);

static int check_desc(const amos_mxfp4_gemm_desc_t* d) {
  if (!d) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  if (d->M < 1 || d->N < 1 || d->K < 1)
    return set_error(AMOS_ERR_BAD_ARG, "4-bit product of extents M %lld, N %lld, K %lld", (long long)d->M, (long long)d->N, (long long)d->K);
  if (d->M >= (int64_t)1 << 30 || d->N >= (int64_t)1 << 30 || d->K >= (int64_t)1 << 31)
    return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: M or N of 2^30 and more, or K of 2^31 and more");
  if (d->a_dtype != AMOS_MXFP4 && !is_dense_dtype(d->a_dtype))
    return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: A of dtype %d (4 bits, fp32, fp16 or bf16)", d->a_dtype);
  if (!is_dense_dtype(d->out_dtype)) return set_error(AMOS_ERR_UNSUPPORTED, "4-bit product: output dtype %d (fp32, fp16 or bf16)", d->out_dtype);
  return 0;
}

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// Dense rows of A are quantised by the few-rows kernel itself where every workgroup can afford to read and convert all of
// them: rows of at most 4096 elements (eight waves of a turn each; the sixteen of K = 8192 come out behind), at most 32 KB
// of them, no more than three rounds of workgroups.  Else by a launch of its own, codes and scales in the workspace.  (On the GPU, fused / apart: 1 x 4096 x 4096 bf16 5.9 / 5.9 us, 8 x 4096 x 2048 4.7 / 5.3,
// 16 x 1024 x 1024 4.4 / 5.0; 1 x 4096 x 8192 9.3 / 8.5, 4 x 4096 x 4096 fp32, 64 KB, 6.8 / 6.2, 1 x 28672 x 8192 54 / 28.  A launch
// and an allocation less are 3 us of the host's time as well.)
static bool quantize_first(const amos_mxfp4_gemm_desc_t* d) {
  if (d->a_dtype == AMOS_MXFP4) return false;
  const bool fused = d->M <= 16 && d->K <= 4096 && d->N <= 768 * 16 && d->M * d->K * dense_size(d->a_dtype) <= 32 << 10;
  return !fused;
}

// Blocks of 16 rows of B times runs of 16 (up to 16 rows of A) or 32 tokens.  Above 16 rows the few-rows kernel is ahead
// while one round takes its blocks (24 x 2048 x 4096: 5.5 us, 32x64 tiles 6.8; 512 x 512 x 4096, two rounds: 7.4 / 6.9);
// the tiled kernels' offsets inside a tile have 32 bits.
struct MxChoice {
  int src;      // what the kernel reads A from (dense rows that are quantised first: SRC_MX)
  int rt, tt;   // few rows: row blocks and token blocks of a workgroup; 0: tiles
  int tile;     // ... of kTiles
};
static MxChoice choose(const amos_mxfp4_gemm_desc_t* d) {
  MxChoice c = {SRC_MX, 0, 0, 0};
  if (d->a_dtype != AMOS_MXFP4 && !quantize_first(d)) c.src = d->a_dtype == AMOS_F32 ? SRC_F32 : d->a_dtype == AMOS_F16 ? SRC_F16 : SRC_BF16;
  const int64_t blocks = (d->N + 15) / 16 * (d->M <= 16 ? 1 : (d->M + 31) / 32);
  const bool far = mx_pitch(d->K) / 64 >= 1 << 16;
  if (c.src != SRC_MX || (d->M <= 16 && (blocks <= 768 || far))) {   // (16384 rows of B: 9.0 us, 32x64 tiles 8.3)
    c.rt = few_blocks(blocks);
    c.tt = 1;
  } else if (blocks <= 256 || far) {
    c.rt = 1;
    c.tt = 2;
  } else {
    c.tile = pick_tile(d->M, d->N);
  }
  return c;
}
template <int SRC>
static int launch_few_blocks(const MxGemmParams& p, int rt, hipStream_t stream) {
  if (rt == 2) return launch_few<SRC, 2, 1>(p, stream);
  if (rt == 3) return launch_few<SRC, 3, 1>(p, stream);
  return launch_few<SRC, 1, 1>(p, stream);
}
static int launch_choice(const MxChoice& c, const MxGemmParams& p, hipStream_t stream) {
  if (c.tt == 2) return launch_few<SRC_MX, 1, 2>(p, stream);
  if (c.tt == 1) {
    if (c.src == SRC_F32) return launch_few_blocks<SRC_F32>(p, c.rt, stream);
    if (c.src == SRC_F16) return launch_few_blocks<SRC_F16>(p, c.rt, stream);
    if (c.src == SRC_BF16) return launch_few_blocks<SRC_BF16>(p, c.rt, stream);
    return launch_few_blocks<SRC_MX>(p, c.rt, stream);
  }
  if (c.tile == 0) return launch_tile<1, 4, 32, 64, 4, true>(p, stream);
  if (c.tile == 1) return launch_tile<2, 2, 64, 64, 4, true>(p, stream);
  if (c.tile == 2) return launch_tile<2, 4, 128, 128, 4, true>(p, stream);
  if (c.tile == 3) return launch_tile<2, 4, 128, 256, 2, true>(p, stream);
  return launch_tile<4, 2, 256, 256, 2, false>(p, stream);
}
static const char* choice_name(const MxChoice& c) {
  static const char* const few[4][3] = {{"amos_mx_gemm_few<mxfp4,1,1>", "amos_mx_gemm_few<mxfp4,2,1>", "amos_mx_gemm_few<mxfp4,3,1>"},
                                        {"amos_mx_gemm_few<f32,1,1>", "amos_mx_gemm_few<f32,2,1>", "amos_mx_gemm_few<f32,3,1>"},
                                        {"amos_mx_gemm_few<f16,1,1>", "amos_mx_gemm_few<f16,2,1>", "amos_mx_gemm_few<f16,3,1>"},
                                        {"amos_mx_gemm_few<bf16,1,1>", "amos_mx_gemm_few<bf16,2,1>", "amos_mx_gemm_few<bf16,3,1>"}};
  static const char* const tile[5] = {"amos_mx_gemm_tile<32x64>", "amos_mx_gemm_tile<64x64>", "amos_mx_gemm_tile<128x128>",
                                      "amos_mx_gemm_tile<128x256>", "amos_mx_gemm_tile<256x256>"};
  return c.tt == 2 ? "amos_mx_gemm_few<mxfp4,1,2>" : c.tt == 1 ? few[c.src][c.rt - 1] : tile[c.tile];
}

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
  const MxChoice c = choose(d);
  if (c.src != SRC_MX) {
    p.dense = A;
  } else if (dense) {
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
  rc = launch_choice(c, p, stream);
  if (rc) return rc;
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(err));
  return 0;
}

}  // namespace amos

using namespace amos;

extern "C" {

size_t amos_mxfp4_gemm_workspace_bytes(const amos_mxfp4_gemm_desc_t* desc) {
  if (check_desc(desc)) return 0;
  if (!quantize_first(desc)) return 0;   // (nothing to keep)
  const int64_t pitch = mx_pitch(desc->K);
  return (size_t)(round256(desc->M * pitch) + round256(desc->M * (pitch / 16)));
}

const char* amos_mxfp4_gemm_kernel_name(const amos_mxfp4_gemm_desc_t* desc) { return check_desc(desc) ? nullptr : choice_name(choose(desc)); }

int amos_mxfp4_gemm(const amos_mxfp4_gemm_desc_t* desc, const amos_mxfp4_epilogue_t* epilogue, const void* A, const void* a_scales,
                    const void* B, const void* b_scales, void* C, void* workspace, size_t ws_bytes, void* stream) {
  return run(desc, epilogue, A, a_scales, B, b_scales, C, workspace, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
