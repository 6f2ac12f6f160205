// Microscaled 4-bit matrices: blocks of 32 consecutive elements of a row share a power-of-two scale.
//
//   codes  [rows][pitch] bytes, pitch = 64 * ceil(cols / 128): two e2m1 codes a byte, the element of
//          the lower index in the low half; elements past `cols` are zeros
//   scales [rows][pitch / 16] bytes: 2^(byte - 127), 255 = not a number; behind the last block 0
//
// A row of codes is a whole number of the 64-byte pieces that one matrix instruction of K = 128
// takes from it, and its scales are whole 32-bit words; where 128 divides cols there is no padding.
//
// For a block with largest magnitude m the scale is 2^e, e = max(floor(log2 m) - 2, -127): it brings
// m into [4, 8), and e2m1 holds 0, 1/2, 1, 3/2, 2, 3, 4, 6; each element is rounded to the nearest
// (ties to the even code), magnitudes above 6 become 6.  In bits: the scale byte is m's exponent field
// less 2, at least 0 (fields 0 to 2, subnormals among them, all give 2^-127).  A block that holds an
// infinity or a NaN gets the scale 255 and stands for NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dense_type.h"

namespace amos {

constexpr int kMxBlock = 32;
__host__ __device__ inline int64_t mx_pitch(int64_t cols) { return (cols + 127) / 128 * 64; }

// scale byte of a block from the largest |bits| among its elements' fp32 patterns
__device__ __forceinline__ unsigned mx_scale_byte(unsigned top_bits) {
  const unsigned field = top_bits >> 23;
  return field == 255 ? 255u : field < 2 ? 0u : field - 2;
}
// eight fp32 values -> eight codes.  The conversion instruction divides by the power of two in the
// exponent field of its scale operand (field 0 = 2^-127), rounds to nearest even and saturates at 6:
// for finite values exactly the definition above (tests/test_gpu_mxfp4_reach.py goes over all scales).
__device__ __forceinline__ unsigned mx_encode8(const float* v, unsigned scale_byte) {
  const float s = __builtin_bit_cast(float, scale_byte << 23);
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
  return scale_byte == 255 ? 0u : c;
}
__device__ __forceinline__ void mx_decode8(unsigned codes, unsigned scale_byte, float* v) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const float s = __builtin_bit_cast(float, scale_byte == 255 ? 127u << 23 : scale_byte << 23);
  v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0);
  v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
  v2f c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2);
  v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  if (scale_byte == 255) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_nanf("");
  }
}
__device__ __forceinline__ unsigned mx_abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

}  // namespace amos
