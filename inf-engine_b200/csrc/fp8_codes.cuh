// From numbers to e4m3 codes and a power of two that scales them: what the quantisers and the product that quantises share.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace {

constexpr int GROUP = 128;             // columns (of a weight: rows too) that share a scale

// 8 numbers of a row as they lie in memory; zeros from column `cols` on
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16* __restrict__ row, int col, int cols, bool vec) {
    if (vec && col + 8 <= cols) {
      u = *reinterpret_cast<const uint4*>(row + col);
    } else if (col + 8 <= cols) {
      // a row that starts anywhere: whole words, and where it starts between two, halves at both ends
      const uint16_t* at = reinterpret_cast<const uint16_t*>(row + col);
      if (((uintptr_t)at & 2) == 0) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(at);
        u = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(at + 1);
        const uint32_t first = at[0], a = w[0], b = w[1], c = w[2], last = at[7];
        u = make_uint4(first | a << 16, __byte_perm(a, b, 0x5432), __byte_perm(b, c, 0x5432), c >> 16 | last << 16);
      }
    } else {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = col + j < cols ? __bfloat16_as_ushort(row[col + j]) : 0;
      u = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* __restrict__ row, int col, int cols, bool vec) {
    if (vec && col + 8 <= cols) {
      a = *reinterpret_cast<const float4*>(row + col);
      b = *reinterpret_cast<const float4*>(row + col + 4);
    } else if (col + 8 <= cols && ((uintptr_t)(row + col) & 7) == 0) {
      const float2* at = reinterpret_cast<const float2*>(row + col);
      const float2 c = at[0], d = at[1], e = at[2], f = at[3];
      a = make_float4(c.x, c.y, d.x, d.y);
      b = make_float4(e.x, e.y, f.x, f.y);
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? row[col + j] : 0.f;
      a = make_float4(v[0], v[1], v[2], v[3]);
      b = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The largest magnitude of 8 numbers on top of m.  A maximum passes a NaN over, so only an infinity shows; a group whose maximum
// is one looks again, number by number.
__device__ __forceinline__ float largest8(const Raw8<float>& r, float m) {
  m = fmaxf(m, fmaxf(fmaxf(fabsf(r.a.x), fabsf(r.a.y)), fmaxf(fabsf(r.a.z), fabsf(r.a.w))));
  return fmaxf(m, fmaxf(fmaxf(fabsf(r.b.x), fabsf(r.b.y)), fmaxf(fabsf(r.b.z), fabsf(r.b.w))));
}
__device__ __forceinline__ float largest8(const Raw8<bf16>& r, float m) {
  const auto two = [](uint32_t u) { u &= 0x7fff7fffu; return *reinterpret_cast<const __nv_bfloat162*>(&u); };
  const __nv_bfloat162 h = __hmax2(__hmax2(two(r.u.x), two(r.u.y)), __hmax2(two(r.u.z), two(r.u.w)));
  return fmaxf(m, fmaxf(__low2float(h), __high2float(h)));
}
template <typename T> __device__ __forceinline__ float largest_finite8(const Raw8<T>& r, float m) {
  float v[8];
  r.get(v);
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

// 8 codes of the numbers times `inverse`, the first in the lowest byte.  A NaN becomes one; an infinity would become 448, so where
// the group has one (`infinite`) it is made a NaN first.
template <typename T> __device__ __forceinline__ uint2 codes8(const Raw8<T>& r, float inverse, bool infinite) {
  float v[8];
  r.get(v);
  if (infinite) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = finite(v[j]) ? v[j] : __uint_as_float(0x7fffffffu);
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * j] * inverse, v[2 * j + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Memory of scales [rows, groups], float32: the larger stride goes from stretch to stretch.
inline Span scales_span(const void* at, long long rows, long long groups, long long s_row, long long s_col) {
  if (rows > 1 && (groups == 1 || s_row >= s_col)) return {(uintptr_t)at, rows, 4 * ((groups - 1) * s_col + 1), 4 * s_row};
  return {(uintptr_t)at, groups, 4 * ((rows - 1) * s_row + 1), 4 * s_col};
}

}  // namespace
