// Element types of the operators that compute in fp32 and hold tensors in fp32, fp16 or bf16: loads
// widen exactly, stores round to nearest even, once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/amos_mi355x.h"

namespace amos {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct TypeF32 {
  typedef float raw_t;
  static constexpr int ES = 4;
  static __device__ __forceinline__ float widen(raw_t v) { return v; }
  static __device__ __forceinline__ raw_t narrow(float v) { return v; }
};
struct TypeF16 {
  typedef _Float16 raw_t;
  static constexpr int ES = 2;
  static __device__ __forceinline__ float widen(raw_t v) { return (float)v; }
  static __device__ __forceinline__ raw_t narrow(float v) { return (_Float16)v; }
};
struct TypeBF16 {
  typedef __bf16 raw_t;
  static constexpr int ES = 2;
  static __device__ __forceinline__ float widen(raw_t v) {
    return __builtin_bit_cast(float, (unsigned)__builtin_bit_cast(unsigned short, v) << 16);
  }
  static __device__ __forceinline__ raw_t narrow(float v) { return (__bf16)v; }
};

// N consecutive elements that are aligned to their own size (or to 16 bytes, if that is less)
template <class T, int N>
struct DenseVec {
  typedef typename T::raw_t raw_t;
  typedef raw_t vec_t __attribute__((ext_vector_type(N)));
  static __device__ __forceinline__ vec_t read(const raw_t* p) { return *(const vec_t*)p; }
  static __device__ __forceinline__ void widen(vec_t x, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = T::widen(x[i]);
  }
  static __device__ __forceinline__ void load(const raw_t* p, float* v) { widen(read(p), v); }
  static __device__ __forceinline__ void store_streaming(raw_t* p, const float* v) {
    vec_t x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = T::narrow(v[i]);
    __builtin_nontemporal_store(x, (vec_t*)p);
  }
  static __device__ __forceinline__ void store(raw_t* p, const float* v) {
    vec_t x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = T::narrow(v[i]);
    *(vec_t*)p = x;
  }
};

// one element of a tensor whose type is known at launch only (vectors of coefficients, fused tails)
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == AMOS_F32) return ((const float*)p)[i];
  if (dtype == AMOS_F16) return TypeF16::widen(((const _Float16*)p)[i]);
  return TypeBF16::widen(((const __bf16*)p)[i]);
}
// N of them in a row, or `otherwise` where there is no tensor: the type is looked at once, the loads
// are in flight together
template <int N>
__device__ __forceinline__ void load_run_any(const void* p, int64_t at, int dtype, float otherwise, float* v) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = otherwise;
  } else if (dtype == AMOS_F32) {
    const float* const q = (const float*)p + at;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = q[i];
  } else {
    const unsigned short* const q = (const unsigned short*)p + at;
    unsigned short raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = q[i];
    if (dtype == AMOS_F16) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = TypeF16::widen(__builtin_bit_cast(_Float16, raw[i]));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = TypeBF16::widen(__builtin_bit_cast(__bf16, raw[i]));
    }
  }
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float v) {
  if (dtype == AMOS_F32) ((float*)p)[i] = v;
  else if (dtype == AMOS_F16) ((_Float16*)p)[i] = TypeF16::narrow(v);
  else ((__bf16*)p)[i] = TypeBF16::narrow(v);
}

inline bool is_dense_dtype(int d) { return d == AMOS_F32 || d == AMOS_F16 || d == AMOS_BF16; }
inline int dense_size(int d) { return d == AMOS_F32 ? 4 : 2; }

}  // namespace amos
