// Quantisation to and from microscaled 4 bits (format: mxfp4.h).  All three kernels move bytes: a
// block's maximum, its scale and its codes are found from registers in one pass over the input.
// 8192 x 8192 bf16 (170 MB in and out; a large copy reaches 5.1 TB/s): along the rows 31 us, 5.5 TB/s; down the columns
// 36 us, 4.7 TB/s; back 26 us, 6.5 TB/s.  fp32 (304 MB): 52, 64 and 62 us.
#include <string.h>

#include "fast_div.h"
#include "mapper.h"
#include "mxfp4.h"

namespace amos {

struct QuantParams {
  const void* x;          // dense matrix
  unsigned char* codes;
  unsigned char* scales;
  int64_t rows;           // of the quantised matrix, in this launch
  int64_t cols;           // ... and the elements of its rows
  int64_t ld;             // elements between rows of x
  int64_t pitch;          // bytes between rows of codes
  FastDiv per_row;        // units of a row of the row kernels
  int units;              // rows * units of a row
};

// Eight elements a lane (16 bytes of a 16-bit type), four neighbouring lanes a block: the block's
// maximum meets over the quad (two DPP steps), the lane's eight codes are one 32-bit store: a wave writes 256
// bytes of codes in one piece.
template <class T>
__global__ __launch_bounds__(256) void amos_mx_quantize_rows(const QuantParams p) {
  const int unit = blockIdx.x * 256 + threadIdx.x;
  if (unit >= p.units) return;   // (units are a multiple of 16: a quad stays or leaves whole)
  const int row = fast_div(unit, p.per_row);
  const int piece = unit - row * (int)(p.pitch / 4);
  const int64_t col = (int64_t)piece * 8;
  const typename T::raw_t* const x = (const typename T::raw_t*)p.x + row * p.ld + col;
  float v[8];
  if (col + 8 <= p.cols) {
    if constexpr (T::ES == 2) {
      DenseVec<T, 8>::load(x, v);
    } else {
      DenseVec<T, 4>::load(x, v);
      DenseVec<T, 4>::load(x + 4, v + 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < p.cols ? T::widen(x[i]) : 0.f;
  }
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned b = mx_abs_bits(v[i]);
    top = b > top ? b : top;
  }
  unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, true);   // lane ^ 1
  top = other > top ? other : top;
  other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, true);            // lane ^ 2
  top = other > top ? other : top;
  const unsigned scale = mx_scale_byte(top);
  *(unsigned*)(p.codes + row * p.pitch + piece * 4) = mx_encode8(v, scale);
  if ((piece & 3) == 0) p.scales[row * (p.pitch / 16) + piece / 4] = (unsigned char)scale;
}

// Blocks down the columns of x: the quantised transpose.  A wave takes 32 rows of 64 columns (a lane
// a column: no exchange for the maximum, a wave's load is 128 or 256 bytes of a row), a workgroup 256 rows, so that a
// column leaves as 128 bytes of codes, one memory line; the columns meet in LDS for that.
template <class T>
__global__ __launch_bounds__(512) void amos_mx_quantize_columns(const QuantParams p) {
  constexpr int CP = 128 + 16;     // bytes of a column in LDS (16 more: neighbouring columns on other banks)
  __shared__ __attribute__((aligned(16))) unsigned char codes[64 * CP];
  __shared__ __attribute__((aligned(8))) unsigned char scales[64 * 8];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t c0 = (int64_t)blockIdx.x * 64, r0 = (int64_t)blockIdx.y * 256;
  const int64_t col = c0 + lane < p.rows ? c0 + lane : p.rows - 1;   // (p.rows = columns of x)
  const int64_t first = r0 + wave * 32;
  float v[32];
  const typename T::raw_t* x = (const typename T::raw_t*)p.x + first * p.ld + col;
  if (first + 32 <= p.cols) {
    typename T::raw_t raw[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) raw[i] = x[i * p.ld];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = T::widen(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = first + i < p.cols ? T::widen(x[i * p.ld]) : 0.f;
  }
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const unsigned b = mx_abs_bits(v[i]);
    top = b > top ? b : top;
  }
  const unsigned scale = mx_scale_byte(top);
  v4u c;
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = mx_encode8(v + 8 * i, scale);
  *(v4u*)(codes + lane * CP + wave * 16) = c;
  scales[lane * 8 + wave] = (unsigned char)scale;
  __syncthreads();
  {
    const int k = t >> 3, part = t & 7;      // eight lanes a column
    const int64_t at = (int64_t)blockIdx.y * 128 + part * 16;
    if (c0 + k < p.rows && at < p.pitch) *(v4u*)(p.codes + (c0 + k) * p.pitch + at) = *(const v4u*)(codes + k * CP + part * 16);
  }
  if (t < 128) {
    const int k = t >> 1, part = t & 1;
    const int64_t at = (int64_t)blockIdx.y * 8 + part * 4;
    if (c0 + k < p.rows && at < p.pitch / 16) *(unsigned*)(p.scales + (c0 + k) * (p.pitch / 16) + at) = *(const unsigned*)(scales + k * 8 + part * 4);
  }
}

template <class T>
__global__ __launch_bounds__(256) void amos_mx_dequantize(const QuantParams p) {
  const int unit = blockIdx.x * 256 + threadIdx.x;
  if (unit >= p.units) return;
  const int row = fast_div(unit, p.per_row);
  const int piece = unit - row * (int)((p.cols + 7) / 8);
  const int64_t col = (int64_t)piece * 8;
  const unsigned c = *(const unsigned*)(p.codes + row * p.pitch + piece * 4);
  const unsigned s = p.scales[row * (p.pitch / 16) + piece / 4];
  float v[8];
  mx_decode8(c, s, v);
  typename T::raw_t* const x = (typename T::raw_t*)p.x + row * p.ld + col;
  if (col + 8 <= p.cols) {
    if constexpr (T::ES == 2) {
      DenseVec<T, 8>::store(x, v);
    } else {
      DenseVec<T, 4>::store(x, v);
      DenseVec<T, 4>::store(x + 4, v + 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < p.cols) x[i] = T::narrow(v[i]);
  }
}

template <class T>
static void launch_rows(const QuantParams& p, bool back, hipStream_t stream) {
  const dim3 grid((unsigned)((p.units + 255) / 256)), block(256);
  if (back) hipLaunchKernelGGL((amos_mx_dequantize<T>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((amos_mx_quantize_rows<T>), grid, block, 0, stream, p);
}
template <class T>
static void launch_columns(const QuantParams& p, unsigned gy, hipStream_t stream) {
  hipLaunchKernelGGL((amos_mx_quantize_columns<T>), dim3((unsigned)((p.rows + 63) / 64), gy), dim3(512), 0, stream, p);
}

static int check_mx_matrix(const amos_mxfp4_desc_t* d, const void* x, const void* codes, const void* scales, const char* what) {
  if (!d || !x || !codes || !scales) return set_error(AMOS_ERR_BAD_ARG, "null pointer argument");
  if (d->rows < 1 || d->cols < 1) return set_error(AMOS_ERR_BAD_ARG, "%s of a %lld x %lld matrix", what, (long long)d->rows, (long long)d->cols);
  if (d->rows >= (int64_t)1 << 31 || d->cols >= (int64_t)1 << 31)
    return set_error(AMOS_ERR_UNSUPPORTED, "%s: extents of 2^31 and more", what);
  if (!is_dense_dtype(d->dtype)) return set_error(AMOS_ERR_UNSUPPORTED, "%s: dtype %d (fp32, fp16 or bf16)", what, d->dtype);
  if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
    return set_error(AMOS_ERR_BAD_ARG, "%s: codes must be 16-byte aligned, scales 4-byte aligned", what);
  if ((uintptr_t)x & (dense_size(d->dtype) - 1)) return set_error(AMOS_ERR_BAD_ARG, "%s: misaligned matrix", what);
  return 0;
}

// launches of the row kernels: as many rows each as keep a launch's units below 2^30
static int run_rows(const amos_mxfp4_desc_t* d, const void* x, void* codes, void* scales, bool back, hipStream_t stream) {
  QuantParams p;
  memset(&p, 0, sizeof(p));
  const int es = dense_size(d->dtype);
  p.cols = p.ld = d->cols;
  p.pitch = mx_pitch(d->cols);
  const int64_t per_row = back ? (d->cols + 7) / 8 : p.pitch / 4;
  p.per_row = make_fast_div((uint32_t)per_row);
  const int64_t most = ((int64_t)1 << 30) / per_row;   // (per_row < 2^28)
  for (int64_t r = 0; r < d->rows; r += most) {
    p.rows = d->rows - r < most ? d->rows - r : most;
    p.units = (int)(p.rows * per_row);
    p.x = (const char*)x + r * p.ld * es;
    p.codes = (unsigned char*)codes + r * p.pitch;
    p.scales = (unsigned char*)scales + r * (p.pitch / 16);
    if (d->dtype == AMOS_F32) launch_rows<TypeF32>(p, back, stream);
    else if (d->dtype == AMOS_F16) launch_rows<TypeF16>(p, back, stream);
    else launch_rows<TypeBF16>(p, back, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  }
  return 0;
}

int mx_quantize(const amos_mxfp4_desc_t* d, const void* x, void* codes, void* scales, hipStream_t stream) {
  int rc = check_mx_matrix(d, x, codes, scales, "quantisation");
  if (rc) return rc;
  if (d->axis == 1) return run_rows(d, x, codes, scales, false, stream);
  if (d->axis != 0) return set_error(AMOS_ERR_BAD_ARG, "quantisation along axis %d of a matrix", d->axis);
  QuantParams p;
  memset(&p, 0, sizeof(p));
  p.cols = d->rows;
  p.ld = d->cols;
  p.pitch = mx_pitch(d->rows);
  const int64_t slabs = (d->rows + 255) / 256;   // of 256 rows of x: the grid's second extent
  if (slabs > 65535) return set_error(AMOS_ERR_UNSUPPORTED, "quantisation along axis 0 of more than %lld rows", 65535LL * 256);
  constexpr int64_t most = (int64_t)1 << 24;     // columns of a launch: a grid has fewer than 2^32 threads
  for (int64_t c = 0; c < d->cols; c += most) {
    p.rows = d->cols - c < most ? d->cols - c : most;
    p.x = (const char*)x + c * dense_size(d->dtype);
    p.codes = (unsigned char*)codes + c * p.pitch;
    p.scales = (unsigned char*)scales + c * (p.pitch / 16);
    if (d->dtype == AMOS_F32) launch_columns<TypeF32>(p, (unsigned)slabs, stream);
    else if (d->dtype == AMOS_F16) launch_columns<TypeF16>(p, (unsigned)slabs, stream);
    else launch_columns<TypeBF16>(p, (unsigned)slabs, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(AMOS_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  }
  return 0;
}

int mx_dequantize(const amos_mxfp4_desc_t* d, const void* codes, const void* scales, void* x, hipStream_t stream) {
  int rc = check_mx_matrix(d, x, codes, scales, "dequantisation");
  if (rc) return rc;
  if (d->axis != 1) return set_error(AMOS_ERR_BAD_ARG, "dequantisation along axis %d (blocks run along the rows: 1)", d->axis);
  return run_rows(d, x, (void*)codes, (void*)scales, true, stream);
}

}  // namespace amos

using namespace amos;

extern "C" {

int64_t amos_mxfp4_pitch(int64_t cols) { return cols < 1 ? 0 : mx_pitch(cols); }

int amos_mxfp4_quantize(const amos_mxfp4_desc_t* desc, const void* x, void* codes, void* scales, void* stream) {
  return mx_quantize(desc, x, codes, scales, (hipStream_t)stream);
}
int amos_mxfp4_dequantize(const amos_mxfp4_desc_t* desc, const void* codes, const void* scales, void* out, void* stream) {
  return mx_dequantize(desc, codes, scales, out, (hipStream_t)stream);
}

}  // extern "C"
