// Product of microscaled 4-bit matrices (format: mxfp4.h) for gfx950:
//   C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]) (+ D[m][n]),  fp32 accumulation, C in fp32, fp16 or bf16.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 4-bit operands with their scales: lane l holds one whole
// block -- the 16 bytes of row l % 16 at K = 32 (l / 16) -- and, in a register of its own, that
// block's scale byte, so a block's scale costs no arithmetic at all.  The accumulator of lane l is
// column l % 16 of rows 4 (l / 16) + r.  A scale byte of 255 makes the sums it enters NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxfp4.h"

namespace amos {

typedef int mx_v4i __attribute__((ext_vector_type(4)));
typedef int mx_v8i __attribute__((ext_vector_type(8)));

struct MxTail {            // what is added to the sums before they are rounded to C's type, once
  const void* bias;        // [N] or null
  const void* add;         // [M][N] or null
  int bias_dtype, add_dtype;
};

struct MxGemmParams {
  const unsigned char* a;  // [M][pitch] codes, or null: `dense`
  const unsigned char* as; // [M][pitch / 16]
  const unsigned char* b;  // [N][pitch]
  const unsigned char* bs;
  const void* dense;       // [M][K] elements that the kernel quantises on their way in
  void* c;                 // [M][N]
  int M, N, K;
  int steps;               // pitch / 64: steps of K = 128
  int out_dtype;
  MxTail tail;
};

// OP: which byte of the scale registers
template <int OP = 0>
__device__ __forceinline__ v4f mx_mfma(mx_v4i a, mx_v4i b, v4f c, int sa, int sb) {
  const mx_v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, OP, sa, OP, sb);
}

__device__ __forceinline__ float mx_tail(const MxTail& t, float v, int64_t m, int n, int N) {
  if (t.bias) v += load_any(t.bias, n, t.bias_dtype);
  if (t.add) v += load_any(t.add, m * N + n, t.add_dtype);
  return v;
}

}  // namespace amos
