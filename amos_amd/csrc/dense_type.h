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

// N consecutive elements of a tensor in global memory, aligned to one element only: the hardware takes 16-byte accesses at
// any address, so rows of any length and views that start anywhere need no kernels of their own
template <class T, int N>
struct DenseVec {
  typedef typename T::raw_t raw_t;
  typedef raw_t vec_t __attribute__((ext_vector_type(N)));
  typedef raw_t mem_t __attribute__((ext_vector_type(N), aligned(T::ES)));
  static __device__ __forceinline__ vec_t read(const raw_t* p) { return *(const mem_t*)p; }
  static __device__ __forceinline__ void widen(vec_t x, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = T::widen(x[i]);
  }
  static __device__ __forceinline__ vec_t narrow(const float* v) {
    vec_t x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = T::narrow(v[i]);
    return x;
  }
  static __device__ __forceinline__ void load(const raw_t* p, float* v) { widen(read(p), v); }
  static __device__ __forceinline__ void store(raw_t* p, const float* v) { *(mem_t*)p = narrow(v); }
  static __device__ __forceinline__ void store_streaming(raw_t* p, const float* v) { __builtin_nontemporal_store(narrow(v), (mem_t*)p); }
};

// one element of a tensor whose type is known at launch only (vectors of coefficients, fused tails)
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == AMOS_F32) return ((const float*)p)[i];
  if (dtype == AMOS_F16) return TypeF16::widen(((const _Float16*)p)[i]);
  return TypeBF16::widen(((const __bf16*)p)[i]);
}
// N of them in a row, or `otherwise` where there is no tensor
template <int N>
__device__ __forceinline__ void load_run_any(const void* p, int64_t at, int dtype, float otherwise, float* v) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = otherwise;
  } else if (dtype == AMOS_F32) {
    DenseVec<TypeF32, N>::load((const float*)p + at, v);
  } else if (dtype == AMOS_F16) {
    DenseVec<TypeF16, N>::load((const _Float16*)p + at, v);
  } else {
    DenseVec<TypeBF16, N>::load((const __bf16*)p + at, v);
  }
}
template <int N>
__device__ __forceinline__ void store_run_any(void* p, int64_t at, int dtype, const float* v) {
  if (dtype == AMOS_F32) DenseVec<TypeF32, N>::store((float*)p + at, v);
  else if (dtype == AMOS_F16) DenseVec<TypeF16, N>::store((_Float16*)p + at, v);
  else DenseVec<TypeBF16, N>::store((__bf16*)p + at, v);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float v) {
  if (dtype == AMOS_F32) ((float*)p)[i] = v;
  else if (dtype == AMOS_F16) ((_Float16*)p)[i] = TypeF16::narrow(v);
  else ((__bf16*)p)[i] = TypeBF16::narrow(v);
}

inline bool is_dense_dtype(int d) { return d == AMOS_F32 || d == AMOS_F16 || d == AMOS_BF16; }
inline int dense_size(int d) { return d == AMOS_F32 ? 4 : 2; }

}  // namespace amos
