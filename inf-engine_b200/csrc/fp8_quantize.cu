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
// Both read every number once and write a byte for it; the HBM rate is the bound: 4,096 rows of 8,192 in bfloat16 take 18.4 us (5.5
// TB/s), in float32 25.7 (6.5), a weight of 16,384 x 2,048 in bfloat16 19.1 us (5.3).  With a look at every number for infinities
// (now only where a group's largest is one) and 8 numbers a lane the bfloat16 rows took 28 us: instructions.
// Rows that do not start on 16 bytes, caches flushed (24.5 and 32.8 us where they do): 4,096 x 8,190 in bfloat16, by words, takes 28.7 us,
// 8,191 (every other row starts between two words) 32.8; in float32, by pairs where a row starts on one, 36.9 and 43.0; number by
// number 38.9 in bfloat16, 49.2 in float32.
#include "fp8_codes.cuh"
#include <numeric>

namespace {

constexpr int QT = 256, BT = 512;      // threads of a block: rows, weights

__device__ __forceinline__ void store8(uint8_t* __restrict__ row, int col, int cols, uint2 c) {
  if (col + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + col) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols) row[col + j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}

// 8 lanes a group, 2 x 8 numbers a lane; U groups of each 8 lanes are under way at once
template <typename T, int U>
__global__ void __launch_bounds__(QT) quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                           float* __restrict__ scales, int rows, int cols, long long ldx,
                                                           long long ldc, long long s_row, long long s_col, int vec) {
  // the product behind this kernel asks for its weights as soon as it starts: it starts when every block here is past the wait, so
  // what wrote them (the block quantiser, perhaps) has finished by then
  pdl_wait();
  pdl_trigger();
  const unsigned per_row = (cols + GROUP - 1) / GROUP, groups = (unsigned)rows * per_row;
  const int lane8 = threadIdx.x & 7;
  const unsigned eight = 0xffu << (threadIdx.x & 24);
  const unsigned g0 = blockIdx.x * (QT / 8 * U) + (threadIdx.x >> 3);
  Raw8<T> raw[U][2];
  unsigned row[U], block[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const unsigned g = min(g0 + i * (QT / 8), groups - 1);          // groups behind the last one: the last again, and not stored
    row[i] = g / per_row;
    block[i] = g - row[i] * per_row;
#pragma unroll
    for (int h = 0; h < 2; ++h) raw[i][h].load(x + row[i] * ldx, block[i] * GROUP + 64 * h + lane8 * 8, cols, vec != 0);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (g0 + i * (QT / 8) >= groups) break;                         // all 8 lanes of a group alike
    float m = largest8(raw[i][1], largest8(raw[i][0], 0.f));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(eight, m, o));
    const bool infinite = !finite(m);
    if (infinite) {
      m = largest_finite8(raw[i][1], largest_finite8(raw[i][0], 0.f));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(eight, m, o));
    }
    const int e = scale_exponent(m);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      store8(codes + row[i] * ldc, block[i] * GROUP + 64 * h + lane8 * 8, cols, codes8(raw[i][h], exp2i(-e), infinite));
    if (lane8 == 0) scales[row[i] * s_row + block[i] * s_col] = exp2i(e);
  }
}

// a block of 128 x 128 a thread block: 16 threads a row, 4 rows a thread, all held in registers between the largest and the codes.
// No trigger ahead of its end: a product behind it may ask for these codes before its wait.
template <typename T>
__global__ void __launch_bounds__(BT) quantize_blocks_kernel(const T* __restrict__ w, uint8_t* __restrict__ codes,
                                                             float* __restrict__ scales, int rows, int cols, long long ldw,
                                                             long long ldc, int vec) {
  constexpr int PER = GROUP * 16 / BT;
  __shared__ float red[33];
  pdl_wait();
  const int col = blockIdx.x * GROUP + (threadIdx.x & 15) * 8;
  const long long row0 = (long long)blockIdx.y * GROUP + (threadIdx.x >> 4);
  Raw8<T> raw[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const long long row = row0 + BT / 16 * i;
    if (row < rows) raw[i].load(w + row * ldw, col, cols, vec != 0);
    else raw[i].zero();
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) m = largest8(raw[i], m);
  m = block_max(m, red);
  const bool infinite = !finite(m);
  if (infinite) {
    m = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) m = largest_finite8(raw[i], m);
    m = block_max(m, red);
  }
  const int e = scale_exponent(m);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const long long row = row0 + BT / 16 * i;
    if (row < rows) store8(codes + row * ldc, col, cols, codes8(raw[i], exp2i(-e), infinite));
  }
  if (threadIdx.x == 0) scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = exp2i(e);
}

#define IE_COINCIDE -7      /* two elements of the scales have one place */
// Whether two elements of [rows, groups] have one place: i s_row = j s_col has its least solution at i = s_col / g, j = s_row / g.
inline bool coincide(long long rows, long long groups, long long s_row, long long s_col) {
  if ((rows > 1 && s_row == 0) || (groups > 1 && s_col == 0)) return rows > 0 && groups > 0;
  if (rows < 2 || groups < 2) return false;
  const long long g = std::gcd(s_row, s_col);
  return s_col / g < rows && s_row / g < groups;
}

// whether rows of x can be read 16 bytes at a time
inline int reads_vectors(const void* x, long long ld, int dtype) {
  return ((uintptr_t)x & 15) == 0 && ld % (dtype == IE_F32 ? 4 : 8) == 0;
}

}  // namespace

// x [rows, cols] (dtype: IE_F32 or IE_BF16, row pitch ldx elements) -> codes [rows, cols] (row pitch ldc bytes, a multiple of 16) and
// scales[row * s_row + group * s_col].  Bytes between the rows of codes are left as they are.
int fp8_quantize_rows(const void* x, int dtype, void* codes, float* scales, int rows, int cols, long long ldx, long long ldc,
                      long long s_row, long long s_col, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return IE_OK;
  if (dtype != IE_F32 && dtype != IE_BF16) return IE_BAD_DTYPE;
  if (((uintptr_t)codes & 15) || ldc % 16) return IE_BAD_ALIGN;
  const int sms = device_sms();
  if (sms <= 0) return IE_BAD_SIZE;
  const long long groups = (long long)rows * ((cols + GROUP - 1) / GROUP);
  if (groups > 0x7fffffffLL) return IE_BAD_SIZE;
  const int vec = reads_vectors(x, ldx, dtype);
  // few groups: one for each 8 lanes, over as many SMs as there are; many: two, so that a thread has four loads under way
  const int u = groups >= 32LL * 8 * sms ? 2 : 1;
  const int grid = (int)((groups + QT / 8 * u - 1) / (QT / 8 * u));
#define IE_ROWS(T, U) launch_k(quantize_rows_kernel<T, U>, grid, QT, 0, stream, (const T*)x, (uint8_t*)codes, scales, rows, cols, ldx, ldc, s_row, s_col, vec)
  if (dtype == IE_F32) return u == 2 ? IE_ROWS(float, 2) : IE_ROWS(float, 1);
  return u == 2 ? IE_ROWS(bf16, 2) : IE_ROWS(bf16, 1);
#undef IE_ROWS
}

// w [rows, cols] -> codes and scales [ceil(rows / 128), ceil(cols / 128)], contiguous
static int fp8_quantize_blocks(const void* w, int dtype, void* codes, float* scales, int rows, int cols, long long ldw, long long ldc,
                               cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return IE_OK;
  if (dtype != IE_F32 && dtype != IE_BF16) return IE_BAD_DTYPE;
  if (((uintptr_t)codes & 15) || ldc % 16) return IE_BAD_ALIGN;
  const dim3 grid((cols + GROUP - 1) / GROUP, (rows + GROUP - 1) / GROUP);
  if (grid.y > 65535) return IE_BAD_SIZE;
  const int vec = reads_vectors(w, ldw, dtype);
  if (dtype == IE_F32)
    return launch_k(quantize_blocks_kernel<float>, grid, BT, 0, stream, (const float*)w, (uint8_t*)codes, scales, rows, cols, ldw, ldc, vec);
  return launch_k(quantize_blocks_kernel<bf16>, grid, BT, 0, stream, (const bf16*)w, (uint8_t*)codes, scales, rows, cols, ldw, ldc, vec);
}

// the entries: arguments as 64-bit words in the order above, which a caller converts in one go; sizes above SIZE_MOST are refused
extern "C" int ie_fp8_quantize_rows(const long long* a) {
  if (beyond(a[4], a[5])) return IE_BAD_SIZE;
  const long long groups = (a[5] + GROUP - 1) / GROUP, size = a[1] == IE_F32 ? 4 : 2;
  const Span scales = scales_span((const void*)a[3], a[4], groups, a[8], a[9]);
  if (overlap(scales, {(uintptr_t)a[2], a[4], a[5], a[7]}) || overlap(scales, {(uintptr_t)a[0], a[4], size * a[5], size * a[6]})) return IE_OVERLAP;
  if (coincide(a[4], groups, a[8], a[9])) return IE_COINCIDE;
  return fp8_quantize_rows((const void*)a[0], (int)a[1], (void*)a[2], (float*)a[3], (int)a[4], (int)a[5], a[6], a[7], a[8], a[9], (cudaStream_t)a[10]);
}
extern "C" int ie_fp8_quantize_blocks(const long long* a) {
  if (beyond(a[4], a[5])) return IE_BAD_SIZE;
  const long long groups = (a[5] + GROUP - 1) / GROUP, size = a[1] == IE_F32 ? 4 : 2;
  const Span scales = scales_span((const void*)a[3], (a[4] + GROUP - 1) / GROUP, groups, groups, 1);
  if (overlap(scales, {(uintptr_t)a[2], a[4], a[5], a[7]}) || overlap(scales, {(uintptr_t)a[0], a[4], size * a[5], size * a[6]})) return IE_OVERLAP;
  return fp8_quantize_blocks((const void*)a[0], (int)a[1], (void*)a[2], (float*)a[3], (int)a[4], (int)a[5], a[6], a[7], (cudaStream_t)a[8]);
}
