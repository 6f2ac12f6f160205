// Tiled product of two microscaled 4-bit matrices: many rows on both sides.
//
// Block tile BI x BJ, K step 256 elements = 128 bytes of every row.  LDS holds NS stages of codes (rows of
// eight 16-byte chunks, XOR-swizzled by row, the swizzle applied on the global side) and two spans of
// scales (32 bytes a row: four K steps).  Both travel by direct copies (global_load_lds, 16 bytes a
// lane; scale rows begin at any word, and rows of fewer than 16 bytes come by words).  A K step is two matrix instructions deep and runs in four phases (half of
// the wave tile's rows, sub-step); the fragments of a phase are read while the one before multiplies.
// The one barrier of a step stands in front of its last phase, where all reads of the stage are
// issued; the copies of the step NS later start behind it, spread over three phases.  A fragment is
// one 16-byte LDS read; its block's scale is a byte of a register that a 2-byte read fills for both
// sub-steps and that the matrix instruction takes as it is: no instruction touches a scale.
// FLAT, where two sets of a step's fragments fit into the registers (all but 256x256): they are read at once, a step ahead
// (2048 x 2048 x 8192, 128x128 tiles with four stages: 25.3 us; in phases, with two, 32.7).
//
// 8192^3, fp32 out: 302 us = 3.6 PFLOP/s (300 - 307 from card to card; bf16 out 293).  Its matrix instructions alone take
// 164 us (6.7 PFLOP/s; a loop of nothing else reaches 7.0 - 7.2 on random operands, 155 us, and 9.2 on zeros: the clock
// goes with the power), with their LDS reads 198 - 203, the copies alone 147 (64 KB a K step and compute unit at 28 bytes
// a cycle, a fifth of it from behind the L2), everything but the stores 238: neither is at its limit by itself (matrix
// cores 42 % busy, LDS 26 %), the two waves of a SIMD do not fill each other's waits.  The 268 MB of results take the rest.
// Tried there: four waves of 128x128 (405 us: one wave a SIMD cannot hide its copies), waves as 2x4 (320); on a faster
// card, on which this kernel took 277 - 281, stores straight from the registers 301, copies in two phases 319.
// Rows past M / N repeat the last one (their sums are not stored).  K is padded to 128 by the format; an
// odd number of 128s ends in a half step whose second half is neither read from memory (its lanes fetch
// the first half again: the row may be the buffer's last) nor multiplied.
#pragma once
#include <type_traits>

#include "igemm_kernel.h"
#include "mxfp4_gemm.h"

namespace amos {

struct MxTileParams {
  MxGemmParams g;
  int tiles_i, tiles_j;
  int vec_scales;       // a row of scales has 16 bytes
  int stream_out;       // an fp32 C larger than the L2s together: written past them (8192^3: 307 -> 302 us)
};

// LDS place of a row's 16-byte chunk.  The swizzle goes by the row inside its block of 16, so that the fragments of
// a wave's row blocks lie at constant distances; a fragment read (16 rows, chunks c and c + 2 in either half of the
// wave) puts two lanes on every 16-byte slot of the 256-byte bank space, its minimum.
__device__ __forceinline__ int mx_lds_offset(int row, int chunk) {
  return row * 128 + ((chunk ^ ((row ^ ((row >> 3) & 1)) & 7)) << 4);
}

#define AMOS_MX_LDS(p) ((__attribute__((address_space(3))) void*)(p))

template <int WI, int WJ, int BI, int BJ, int NS, bool FLAT>
__global__ __launch_bounds__(64 * WI * WJ) void amos_mx_gemm_tile(const MxTileParams t) {
  constexpr int NW = WI * WJ;
  constexpr int TI = BI / (16 * WI), TJ = BJ / (16 * WJ);
  constexpr int HA = TI / 2;
  static_assert(TI % 2 == 0 && TI * WI * 16 == BI && TJ * WJ * 16 == BJ && TJ >= 1, "wave tile");
  constexpr int OPER = BI * 128, STAGE = (BI + BJ) * 128;        // one stage of codes
  constexpr int SCALES = NS * STAGE, SPAN = (BI + BJ) * 32;      // behind them: two spans (four K steps) of scales
  constexpr int QA = BI / 8;
  constexpr int CH = (BI + BJ) / 8 / NW;                         // 1 KB copies of a wave and K step
  constexpr int SG = (BI + BJ) / 32, SV = (SG + NW - 1) / NW;     // copies of scales of a span, of a wave: 16 bytes a lane
  constexpr int SW = CH;                                         // ... of a wave, 4 bytes a lane
  static_assert(CH >= 1 && CH * NW * 8 == BI + BJ && BI % 32 == 0 && BJ % 32 == 0, "copies");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const MxGemmParams& p = t.g;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ;
  int tile_i, tile_j;
  block_to_tile(blockIdx.x, gridDim.x, t.tiles_i, t.tiles_j, tile_i, tile_j);
  const int bi0 = tile_i * BI, bj0 = tile_j * BJ;
  const int64_t pitch = (int64_t)p.steps * 64, spitch = (int64_t)p.steps * 4;
  const unsigned char* const abase = p.a + bi0 * pitch;
  const unsigned char* const bbase = p.b + bj0 * pitch;
  const unsigned char* const asbase = p.as + bi0 * spitch;
  const unsigned char* const bsbase = p.bs + bj0 * spitch;
  // whole K steps, and whether a half one follows
  const int full = p.steps >> 1, half = p.steps & 1, KT = full + half;

  unsigned g_off[CH];
  const int chunk = (lane & 7) ^ (((lane >> 3) ^ (wave & 1)) & 7);   // (NW even: the same for every copy of the wave)
  static_assert(NW % 2 == 0 && QA % 2 == 0, "one swizzle term per wave");
#pragma unroll
  for (int u = 0; u < CH; ++u) {
    const int q = wave + NW * u;
    const int row = (q < QA ? q : q - QA) * 8 + (lane >> 3);
    const int r = q < QA ? (bi0 + row < p.M ? row : p.M - 1 - bi0) : (bj0 + row < p.N ? row : p.N - 1 - bj0);
    g_off[u] = (unsigned)r * (unsigned)pitch + chunk * 16;
  }
  const unsigned back = chunk >= 4 ? 64 : 0;   // what a half step's second half steps back
  // Copies as assembly: behind the builtin the compiler lets every later LDS read wait for all LDS reads before it.
  // The wait states are those of an address register pair that a vector instruction may have written (5) and of M0 (1).
  const unsigned lds0 = (unsigned)(uintptr_t)AMOS_MX_LDS(smem);
  auto issue_copy = [&](int kt, int stage, int u) {
    const int q = wave + NW * u;
    const unsigned char* const base = (q < QA ? abase : bbase) + (int64_t)kt * 128;
    const unsigned off = g_off[u] - (kt >= full ? back : 0u);
    asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds0 + stage * STAGE + q * 1024), "v"(off), "s"(base) : "memory");
  };
  // Scales: a row's 32 bytes of four K steps at once (8 bytes a row and step would touch as many memory lines per
  // step as the codes do).  Bit 3 of the row swaps the two 16-byte halves of its place: sixteen rows on different
  // banks.  A row whose length is no multiple of 16 ends in its last 16 bytes once more: scale_at() reads that much
  // further on.
  auto scale_row = [&](int row) -> unsigned {   // row of the tile (A's, then B's) -> row of its operand, from the tile's first on
    return (unsigned)(row < BI ? (bi0 + row < p.M ? row : p.M - 1 - bi0) : (bj0 + row - BI < p.N ? row - BI : p.N - 1 - bj0));
  };
  auto scale_vec = [&](int span, int u) {      // 32 rows, two lanes a row
    const int first = (wave + NW * u) * 32, row = first + (lane >> 1);
    if (SG % NW && first >= BI + BJ) return;
    const int want = span * 32 + ((lane ^ (row >> 3)) & 1) * 16;
    const unsigned r = scale_row(row);
    const int last = (int)spitch - 16;
    const unsigned off = r * (unsigned)spitch + (unsigned)(want < last ? want : last);
    const unsigned char* const sb = first < BI ? asbase : bsbase;
    asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds0 + SCALES + (span & 1) * SPAN + first * 32), "v"(off), "s"(sb) : "memory");
  };
  auto scale_word = [&](int u) {               // 8 rows, eight lanes a row (the words behind its end: the last one, not used)
    const int first = (wave + NW * u) * 8, row = first + (lane >> 3);
    const int want = (lane & 7) ^ (((row >> 3) & 1) << 2);
    const unsigned r = scale_row(row);
    const int last = p.steps - 1;
    const unsigned off = r * (unsigned)spitch + (unsigned)(want < last ? want : last) * 4;
    const unsigned char* const sb = first < BI ? asbase : bsbase;
    asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds0 + SCALES + first * 32), "v"(off), "s"(sb) : "memory");
  };
  // the next span's scales, in the first step of a span: the copies that follow them until their use are more than the
  // waits below leave in flight.  (A second span has rows of 32 bytes and more behind it.)
  auto issue_scales = [&](int kt) {
    const int span = (kt >> 2) + 1;
    if (span * 4 >= KT || (kt & 3)) return;
#pragma unroll
    for (int u = 0; u < SV; ++u) scale_vec(span, u);
  };

  // Which of a K step's eight blocks a lane group takes is free as long as both operands agree: group q takes blocks
  // 2q and 2q + 1, whose scales are the two bytes of one read.  (A half step has four blocks: block q.)
  const int frag_row = lane & 15, frag_q = lane >> 4;
  const int arow = wi * TI * 16 + frag_row, brow = wj * TJ * 16 + frag_row;
  const int a_off = mx_lds_offset(arow, 2 * frag_q), b_off = OPER + mx_lds_offset(brow, 2 * frag_q);
  const int swap = ((frag_row >> 3) & 1) * 16;
  const int as_off = arow * 32 + 2 * frag_q + swap, bs_off = (BI + brow) * 32 + 2 * frag_q + swap;
  // LDS address of step kt's scale bytes for a row whose place is `off`
  auto scale_at = [&](int off, int kt, bool used) {
    const int ahead = t.vec_scales && used ? (kt >> 1) * 16 + 16 - (int)spitch : 0;   // the last 16 bytes begin earlier by so much
    return smem + SCALES + ((kt >> 2) & 1) * SPAN + (off ^ (((kt >> 1) & 1) * 16)) + (kt & 1) * 8 + (ahead > 0 ? ahead : 0);
  };

  v4f acc[TI][TJ];
#pragma unroll
  for (int a = 0; a < TI; ++a)
#pragma unroll
    for (int b = 0; b < TJ; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};

  constexpr std::integral_constant<int, 0> I0{};
  constexpr std::integral_constant<int, 1> I1{};
  auto first_scales = [&]() {
    if (t.vec_scales) {
#pragma unroll
      for (int u = 0; u < SV; ++u) scale_vec(0, u);
    } else {
#pragma unroll
      for (int u = 0; u < SW; ++u) scale_word(u);
    }
  };
  int st = 0;   // this step's stage
  if constexpr (FLAT) {
    // All fragments of a step are read at once, a step ahead, into a second set of registers: what hides an LDS read
    // is a step's matrix instructions, not a phase's.
    mx_v4i fa[2][2][TI], fb[2][2][TJ];
    int xa[2][TI], xb[2][TJ];
    auto read_all = [&](int kt, int stage, auto set) {
      const char* s = smem + stage * STAGE;
      const char *sa = scale_at(as_off, kt, kt < full), *sb = scale_at(bs_off, kt, kt < full);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int a = 0; a < TI; ++a) fa[set][ks][a] = *(const mx_v4i*)(s + (a_off ^ (ks * 16)) + a * 2048);
#pragma unroll
        for (int b = 0; b < TJ; ++b) fb[set][ks][b] = *(const mx_v4i*)(s + (b_off ^ (ks * 16)) + b * 2048);
      }
#pragma unroll
      for (int a = 0; a < TI; ++a) xa[set][a] = *(const unsigned short*)(sa + a * 512);
#pragma unroll
      for (int b = 0; b < TJ; ++b) xb[set][b] = *(const unsigned short*)(sb + b * 512);
    };
    auto step = [&](int kt, auto set, auto other) {
      const int next = st + 1 == NS ? 0 : st + 1, after = kt + NS < KT ? kt + NS : KT - 1;
      // this wave's copies of the next step have landed (those of the NS - 2 steps behind it may be under way; copies of
      // one width complete in their order) and its reads of this one too: behind the barrier the next stage is whole and
      // this one is free
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * CH) : "memory");
      asm volatile("s_barrier" ::: "memory");
      read_all(kt + 1, next, other);   // (behind the last step: read and not used)
      __builtin_amdgcn_sched_barrier(0);
      issue_scales(kt);
#pragma unroll
      for (int u = 0; u < CH; ++u) issue_copy(after, st, u);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = mx_mfma<0>(fa[set][0][a], fb[set][0][b], acc[a][b], xa[set][a], xb[set][b]);
#pragma unroll
      for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = mx_mfma<1>(fa[set][1][a], fb[set][1][b], acc[a][b], xa[set][a], xb[set][b]);
      __builtin_amdgcn_sched_barrier(0);
      st = next;
    };
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int u = 0; u < CH; ++u) issue_copy(s < KT ? s : KT - 1, s, u);
      if (s == 0) first_scales();
    }
    if (t.vec_scales) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * CH) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    read_all(0, 0, I0);
    int kt = 0;
    for (; kt + 1 < full; kt += 2) {
      step(kt, I0, I1);
      step(kt + 1, I1, I0);
    }
    if (kt < full) step(kt, I0, I1);
  } else {
    static_assert(NS == 2, "LDS takes two stages of the one tile that comes here");
    mx_v4i af[2][HA], bf[2][TJ];      // A: by half of the wave tile's rows; B: by sub-step
    int ax[TI], bx[TJ], bx_next[TJ];   // scales: a register serves both sub-steps
    auto read_a = [&](int kt, int stage, auto h, auto ks) {
      const char* s = smem + stage * STAGE;
      const char* x = scale_at(as_off, kt, kt < full);
#pragma unroll
      for (int a = 0; a < HA; ++a) {
        af[h][a] = *(const mx_v4i*)(s + (a_off ^ (ks * 16)) + (h * HA + a) * 2048);
        if (ks == 0) ax[h * HA + a] = *(const unsigned short*)(x + (h * HA + a) * 512);
      }
    };
    auto read_b = [&](int kt, int stage, auto ks, int* to) {
      const char* s = smem + stage * STAGE;
      const char* x = scale_at(bs_off, kt, kt < full);
#pragma unroll
      for (int b = 0; b < TJ; ++b) {
        bf[ks][b] = *(const mx_v4i*)(s + (b_off ^ (ks * 16)) + b * 2048);
        if (ks == 0) to[b] = *(const unsigned short*)(x + b * 512);
      }
    };
    // One phase: the matrix instructions of half h of sub-step ks, and between them a share of the copies of step kt (a
    // copy keeps its wave from issuing for some 64 cycles: spread out, the matrix core works through them).  The fences
    // keep the compiler from moving the reads in front of a phase down to their use.
    constexpr int SLOTS = 3 * TJ;   // places behind a group of HA instructions in the three phases that carry copies
    auto phase = [&](auto h, auto ks, int part, int kt, int stage) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < TJ; ++b) {
#pragma unroll
        for (int a = 0; a < HA; ++a) acc[h * HA + a][b] = mx_mfma<ks>(af[h][a], bf[ks][b], acc[h * HA + a][b], ax[h * HA + a], bx[b]);
        if (part >= 0) {
          const int slot = part * TJ + b;
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = slot * CH / SLOTS; u < (slot + 1) * CH / SLOTS; ++u) issue_copy(kt, stage, u);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int FIRST = TJ * CH / SLOTS;   // copies of part 0

    // the first NS - 1 steps whole, of the next one the part that otherwise leaves in the step before
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
#pragma unroll
      for (int u = 0; u < CH; ++u) issue_copy(s < KT ? s : KT - 1, s, u);
      if (s == 0) first_scales();
    }
#pragma unroll
    for (int u = 0; u < FIRST; ++u) issue_copy(NS - 1 < KT ? NS - 1 : KT - 1, NS - 1, u);
    if (t.vec_scales) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * CH + FIRST) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    read_a(0, 0, I0, I0);
    read_b(0, 0, I0, bx);

    int last = NS - 1;   // the stage whose copies are under way
    for (int kt = 0; kt < full; ++kt) {
      const int next = st + 1 == NS ? 0 : st + 1;
      const int ahead = kt + NS - 1 < KT ? kt + NS - 1 : KT - 1, after = kt + NS < KT ? kt + NS : KT - 1;
      read_a(kt, st, I1, I0);
      phase(I0, I0, 1, ahead, last);
      issue_scales(kt);
      read_a(kt, st, I0, I1);
      read_b(kt, st, I1, bx);
      phase(I1, I0, 2, ahead, last);
      read_a(kt, st, I1, I1);
      phase(I0, I1, -1, 0, 0);
      // all reads of this stage are issued; once they and this wave's copies of the next step are done (those of the NS - 2
      // steps behind it may be under way), meet: behind the barrier the next stage is whole and this one is free.  (Copies
      // of one width complete in their order.)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * CH) : "memory");
      asm volatile("s_barrier" ::: "memory");
      read_a(kt + 1, next, I0, I0);   // (behind the last step: read and not used)
      read_b(kt + 1, next, I0, bx_next);
      phase(I1, I1, 0, after, st);
#pragma unroll
      for (int b = 0; b < TJ; ++b) bx[b] = bx_next[b];
      last = st;
      st = next;
    }
  }
  if (half) {   // four blocks, one for each lane group
    const char* s = smem + st * STAGE;
    const int ah = mx_lds_offset(arow, frag_q), bh = OPER + mx_lds_offset(brow, frag_q);
    const char *axh = scale_at(as_off - frag_q, full, true), *bxh = scale_at(bs_off - frag_q, full, true);   // (byte q, not 2q)
    mx_v4i g[TJ];
    int y[TJ];
#pragma unroll
    for (int b = 0; b < TJ; ++b) {
      g[b] = *(const mx_v4i*)(s + bh + b * 2048);
      y[b] = *(const unsigned char*)(bxh + b * 512);
    }
#pragma unroll
    for (int a = 0; a < TI; ++a) {
      const mx_v4i f = *(const mx_v4i*)(s + ah + a * 2048);
      const int x = *(const unsigned char*)(axh + a * 512);
#pragma unroll
      for (int b = 0; b < TJ; ++b) acc[a][b] = mx_mfma(f, g[b], acc[a][b], x, y[b]);
    }
  }

  // ---- the sums leave through a strip of LDS per wave (half the wave tile's rows at a time): whole rows, 16 bytes
  // a lane; bias and D join there, in fp32, before the one rounding
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (the last copies have landed, all reads are done)
  constexpr int SP = TJ * 16 + 4, SR = HA * 16;
  static_assert(NW * SR * SP * 4 <= SCALES + 2 * SPAN, "output strip");
  float* const strip = (float*)smem + wave * (SR * SP);
  const int wj0 = bj0 + wj * TJ * 16;
  // V neighbouring results of a lane
  auto emit = [&](int i, int j, const float* from, auto width) {
    constexpr int V = decltype(width)::value;
    float v[V], e[V];
#pragma unroll
    for (int x = 0; x < V; x += 4) {
      const v4f w = *(const v4f*)(from + x);
#pragma unroll
      for (int y = 0; y < 4; ++y) v[x + y] = w[y];
    }
    const int64_t at = (int64_t)i * p.N + j;
    if (i >= p.M || j >= p.N) return;
    if (j + V <= p.N) {
      if (p.tail.bias) {
        load_run_any<V>(p.tail.bias, j, p.tail.bias_dtype, 0.f, e);
#pragma unroll
        for (int x = 0; x < V; ++x) v[x] += e[x];
      }
      if (p.tail.add) {
        load_run_any<V>(p.tail.add, at, p.tail.add_dtype, 0.f, e);
#pragma unroll
        for (int x = 0; x < V; ++x) v[x] += e[x];
      }
      if constexpr (V == 4) {
        if (t.stream_out) DenseVec<TypeF32, 4>::store_streaming((float*)p.c + at, v);
        else DenseVec<TypeF32, 4>::store((float*)p.c + at, v);
      } else {
        if (p.out_dtype == AMOS_F16) DenseVec<TypeF16, 8>::store((_Float16*)p.c + at, v);
        else DenseVec<TypeBF16, 8>::store((__bf16*)p.c + at, v);
      }
    } else {
#pragma unroll
      for (int x = 0; x < V; ++x)
        if (j + x < p.N) store_any(p.c, at + x, p.out_dtype, mx_tail(p.tail, v[x], i, j + x, p.N));
    }
  };
  auto store_half = [&](int h) {
#pragma unroll
    for (int a = 0; a < HA; ++a)
#pragma unroll
      for (int b = 0; b < TJ; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) strip[(a * 16 + 4 * frag_q + r) * SP + b * 16 + frag_row] = acc[h * HA + a][b][r];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int i0 = bi0 + (wi * TI + h * HA) * 16;
    if (p.out_dtype == AMOS_F32) {
      constexpr int LPR = TJ * 4, RPI = 64 / LPR < SR ? 64 / LPR : SR;   // lanes of a row, rows of an instruction
      static_assert(SR % RPI == 0, "strip rows");
#pragma unroll 2
      for (int n = 0; n < SR / RPI; ++n) {
        const int row = n * RPI + lane / LPR, col = (lane % LPR) * 4;
        if (LPR * RPI == 64 || lane < LPR * RPI) emit(i0 + row, wj0 + col, strip + row * SP + col, std::integral_constant<int, 4>{});
      }
    } else {
      constexpr int LPR = TJ * 2, RPI = 64 / LPR < SR ? 64 / LPR : SR;
      static_assert(SR % RPI == 0, "strip rows");
#pragma unroll 2
      for (int n = 0; n < SR / RPI; ++n) {
        const int row = n * RPI + lane / LPR, col = (lane % LPR) * 8;
        if (LPR * RPI == 64 || lane < LPR * RPI) emit(i0 + row, wj0 + col, strip + row * SP + col, std::integral_constant<int, 8>{});
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the strip is read before it is written again)
  };
  store_half(0);
  store_half(1);
}

}  // namespace amos
