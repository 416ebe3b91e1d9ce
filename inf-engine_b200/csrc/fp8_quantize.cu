// Quantising to 8-bit floating point (e4m3) with a scale for each group of 128 numbers: rows (activations; a group is 128
// columns of one row) and weights (a group is a block of 128 rows x 128 columns).
//
//   largest = max |x| over the group's finite numbers
//   scale   = 2^ceil(log2(largest / 448)), at least 2^-126; 1 for a group of zeros
//   code    = e4m3(x / scale), round to nearest even; a number that is not finite becomes NaN (e4m3 has no infinity)
//
// The scale is a power of two on purpose: x / scale is then exact, so a code is ONE rounding of x (half a step of 2^-3
// relative: 2^-4), whichever way the quotient is computed.  A largest / 448 that is no power of two would gain nothing but
// the last binade's top (448 is used to between 0.5 and 1) and cost a second rounding.
//
// Both read every number once and write a byte for it; the HBM rate is the bound.
#include "common.cuh"
#include <cuda_fp8.h>

namespace {

constexpr int GROUP = 128;
constexpr int QT = 256;

// 8 numbers of a row from column `col` (zeros from `cols` on)
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int col, int cols, bool vec, float (&v)[8]) {
  if (vec && col + 8 <= cols) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + col);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const float4 a = *reinterpret_cast<const float4*>(row + col), b = *reinterpret_cast<const float4*>(row + col + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? to_f32(row[col + j]) : 0.f;
  }
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

__device__ __forceinline__ float largest8(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, finite(v[j]) ? fabsf(v[j]) : 0.f);
  return m;
}

// the scale's exponent: 448 = 1.75 * 2^8, so a largest number f * 2^e (1 <= f < 2) takes e - 8, or e - 7 when f > 1.75.  A
// subnormal reads as e = -127 and takes the least exponent either way.
__device__ __forceinline__ int scale_exponent(float largest) {
  const uint32_t u = __float_as_uint(largest);
  if (u == 0) return 0;
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// 8 codes of v / 2^e, the first in the lowest byte
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inverse) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 p;
    p.x = finite(v[2 * j]) ? v[2 * j] * inverse : __uint_as_float(0x7fffffffu);
    p.y = finite(v[2 * j + 1]) ? v[2 * j + 1] * inverse : __uint_as_float(0x7fffffffu);
    w[j] = __nv_cvt_float2_to_fp8x2(p, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

__device__ __forceinline__ void store8(uint8_t* __restrict__ row, int col, int cols, uint2 c) {
  if (col + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + col) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols) row[col + j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}

// 16 lanes a group, 8 numbers a lane
template <typename T>
__global__ void __launch_bounds__(QT) quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                           float* __restrict__ scales, int rows, int cols, long long ldx,
                                                           long long ldc, long long s_row, long long s_col, int vec) {
  pdl_trigger();
  pdl_wait();
  const int per_row = (cols + GROUP - 1) / GROUP;
  const long long groups = (long long)rows * per_row;
  const int lane16 = threadIdx.x & 15;
  for (long long g = (long long)blockIdx.x * (QT / 16) + (threadIdx.x >> 4); g < groups; g += (long long)gridDim.x * (QT / 16)) {
    const long long row = g / per_row;
    const int b = (int)(g - row * per_row), col = b * GROUP + lane16 * 8;
    float v[8];
    load8(x + row * ldx, col, cols, vec != 0, v);
    float m = largest8(v);
    const unsigned half = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(half, m, o));
    const int e = scale_exponent(m);
    store8(codes + row * ldc, col, cols, codes8(v, exp2i(-e)));
    if (lane16 == 0) scales[row * s_row + b * s_col] = exp2i(e);
  }
}

// a block of 128 x 128 a thread block: 16 threads a row, 8 rows a thread, all held in registers between the largest and the codes
template <typename T>
__global__ void __launch_bounds__(QT) quantize_blocks_kernel(const T* __restrict__ w, uint8_t* __restrict__ codes,
                                                             float* __restrict__ scales, int rows, int cols, long long ldw,
                                                             long long ldc, int vec) {
  __shared__ float red[33];
  pdl_trigger();
  pdl_wait();
  const int col = blockIdx.x * GROUP + (threadIdx.x & 15) * 8;
  const long long row0 = (long long)blockIdx.y * GROUP + (threadIdx.x >> 4);
  float v[8][8], m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long row = row0 + 16 * i;
    if (row < rows) {
      load8(w + row * ldw, col, cols, vec != 0, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, largest8(v[i]));
  const int e = scale_exponent(block_max(m, red));
  const float inverse = exp2i(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long row = row0 + 16 * i;
    if (row < rows) store8(codes + row * ldc, col, cols, codes8(v[i], inverse));
  }
  if (threadIdx.x == 0) scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = exp2i(e);
}

// whether rows of x can be read 16 bytes at a time
inline int reads_vectors(const void* x, long long ld, int dtype) {
  return ((uintptr_t)x & 15) == 0 && ld % (dtype == IE_F32 ? 4 : 8) == 0;
}

}  // namespace

// x [rows, cols] (dtype: IE_F32 or IE_BF16, row pitch ldx elements) -> codes [rows, cols] (row pitch ldc bytes, a multiple of 16) and
// scales[row * s_row + group * s_col].  Bytes between the rows of codes are left as they are.
extern "C" int ie_fp8_quantize_rows(const void* x, int dtype, void* codes, float* scales, int rows, int cols, long long ldx,
                                    long long ldc, long long s_row, long long s_col, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return IE_OK;
  if (dtype != IE_F32 && dtype != IE_BF16) return IE_BAD_DTYPE;
  if (((uintptr_t)codes & 15) || ldc % 16) return IE_BAD_ALIGN;
  const int sms = device_sms();
  if (sms <= 0) return IE_BAD_SIZE;
  const long long groups = (long long)rows * ((cols + GROUP - 1) / GROUP), blocks = (groups + QT / 16 - 1) / (QT / 16);
  const int grid = (int)(blocks < 8LL * sms ? blocks : 8LL * sms);
  const int vec = reads_vectors(x, ldx, dtype);
  if (dtype == IE_F32)
    return launch_k(quantize_rows_kernel<float>, grid, QT, 0, stream, (const float*)x, (uint8_t*)codes, scales, rows, cols, ldx, ldc,
                    s_row, s_col, vec);
  return launch_k(quantize_rows_kernel<bf16>, grid, QT, 0, stream, (const bf16*)x, (uint8_t*)codes, scales, rows, cols, ldx, ldc,
                  s_row, s_col, vec);
}

// w [rows, cols] -> codes and scales [ceil(rows / 128), ceil(cols / 128)], contiguous
extern "C" int ie_fp8_quantize_blocks(const void* w, int dtype, void* codes, float* scales, int rows, int cols, long long ldw,
                                      long long ldc, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return IE_OK;
  if (dtype != IE_F32 && dtype != IE_BF16) return IE_BAD_DTYPE;
  if (((uintptr_t)codes & 15) || ldc % 16) return IE_BAD_ALIGN;
  const dim3 grid((cols + GROUP - 1) / GROUP, (rows + GROUP - 1) / GROUP);
  if (grid.y > 65535) return IE_BAD_SIZE;
  const int vec = reads_vectors(w, ldw, dtype);
  if (dtype == IE_F32)
    return launch_k(quantize_blocks_kernel<float>, grid, QT, 0, stream, (const float*)w, (uint8_t*)codes, scales, rows, cols, ldw, ldc, vec);
  return launch_k(quantize_blocks_kernel<bf16>, grid, QT, 0, stream, (const bf16*)w, (uint8_t*)codes, scales, rows, cols, ldw, ldc, vec);
}
