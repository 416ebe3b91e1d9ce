// y[M, N] = x[M, K] w[N, K]^T with both operands in 8-bit floating point (e4m3): x with a scale for each row and 128 columns,
// w with a scale for each block of 128 x 128,
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b]  sum_{k in block b} x[m, k] w[n, k]
//
// inner and outer sums in float32, one rounding to the output's type.
#include "common.cuh"
#include <cuda_fp8.h>

namespace {

constexpr int GROUP = 128;
enum { IE_E4M3 = 2 };      // dtype code of an operand that is quantised already

struct Fp8Params {
  const uint8_t* x;
  const float* sx;
  const uint8_t* w;
  const float* sw;
  void* y;
  int M, N, K;
  long long ldx, sx_row, sx_col, ldw, ldy;
  int y_bf16;
};

__device__ __forceinline__ float code_value(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// tiles of 32 x 32 results, one block of 32 columns at a time through shared memory
__global__ void __launch_bounds__(256) gemm_fp8_kernel(Fp8Params p) {
  __shared__ float xs[32][33], ws[32][33];
  pdl_trigger();
  pdl_wait();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, kb = (p.K + GROUP - 1) / GROUP;
  const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 32, n = n0 + tx;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < kb; ++b) {
    float in[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = b * GROUP; k0 < min(p.K, (b + 1) * GROUP); k0 += 32) {
      __syncthreads();
      for (int i = ty; i < 32; i += 8) {
        xs[i][tx] = (m0 + i < p.M && k0 + tx < p.K) ? code_value(p.x[(m0 + i) * p.ldx + k0 + tx]) : 0.f;
        ws[i][tx] = (n0 + i < p.N && k0 + tx < p.K) ? code_value(p.w[(n0 + i) * p.ldw + k0 + tx]) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k)
        for (int i = 0; i < 4; ++i) in[i] += xs[ty + 8 * i][k] * ws[tx][k];
    }
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + ty + 8 * i;
      if (m < p.M && n < p.N) acc[i] += p.sx[m * p.sx_row + b * p.sx_col] * p.sw[(long long)(n / GROUP) * kb + b] * in[i];
    }
  }
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 8 * i;
    if (m >= p.M || n >= p.N) continue;
    if (p.y_bf16) ((bf16*)p.y)[m * p.ldy + n] = __float2bfloat16_rn(acc[i]);
    else ((float*)p.y)[m * p.ldy + n] = acc[i];
  }
}

}  // namespace

// fp8_quantize.cu
extern "C" int ie_fp8_quantize_rows(const void* x, int dtype, void* codes, float* scales, int rows, int cols, long long ldx,
                                    long long ldc, long long s_row, long long s_col, cudaStream_t stream);

// bytes of scratch that the product of unquantised rows takes: their codes, then their scales [K / 128][M]
extern "C" long long ie_gemm_fp8_scratch(int M, int K) {
  if (M <= 0 || K <= 0) return 0;
  return (long long)M * ((K + 15) / 16 * 16) + 4LL * M * ((K + GROUP - 1) / GROUP);
}

// x: codes (x_dtype IE_E4M3, with sx) or float32 / bfloat16 rows, which are quantised into scratch first
extern "C" int ie_gemm_fp8(const void* x, int x_dtype, const float* sx, const void* w, const float* sw, void* y, int y_dtype, int M,
                           int N, int K, long long ldx, long long sx_row, long long sx_col, long long ldw, long long ldy,
                           void* scratch, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return IE_OK;
  if (K <= 0) return IE_BAD_SIZE;
  if (y_dtype != IE_F32 && y_dtype != IE_BF16) return IE_BAD_DTYPE;
  if (((uintptr_t)w & 15) || ldw % 16) return IE_BAD_ALIGN;
  if (x_dtype != IE_E4M3) {
    if (scratch == nullptr || ((uintptr_t)scratch & 15)) return IE_BAD_ALIGN;
    const long long pitch = (K + 15) / 16 * 16;
    float* scales = reinterpret_cast<float*>((char*)scratch + M * pitch);
    const int rc = ie_fp8_quantize_rows(x, x_dtype, scratch, scales, M, K, ldx, pitch, 1, M, stream);
    if (rc) return rc;
    x = scratch; ldx = pitch; sx = scales; sx_row = 1; sx_col = M;
  }
  if (((uintptr_t)x & 15) || ldx % 16) return IE_BAD_ALIGN;
  Fp8Params p;
  p.x = (const uint8_t*)x; p.sx = sx; p.w = (const uint8_t*)w; p.sw = sw; p.y = y; p.M = M; p.N = N; p.K = K;
  p.ldx = ldx; p.sx_row = sx_row; p.sx_col = sx_col; p.ldw = ldw; p.ldy = ldy; p.y_bf16 = y_dtype == IE_BF16;
  const dim3 grid((N + 31) / 32, (M + 31) / 32);
  if (grid.y > 65535) return IE_BAD_SIZE;
  return launch_k(gemm_fp8_kernel, grid, 256, 0, stream, p);
}
