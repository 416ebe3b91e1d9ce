// What every request has said so far, kept on the device in the request's slot, and logits adjusted by it.
//
//   counts  int32 [slots, vocab]             how often the request generated a token
//   seen    int32 words [slots, ceil(vocab / 32)]   bit t % 32 of word t / 32: the token is in its prompt or was generated
//
// A reset clears slots, an append adds tokens; all updates are whole numbers, so their order does not matter and a call gives
// the same state on every run, tokens and slots that come twice included.
//
// The logits of a row, with s its slot and (r, p, f) its penalties:
//   v = logit[t];   seen[s, t]:  v = v < 0 ? v r : v / r;   counts[s, t] = c > 0:  v -= f c + p
//   v += the row's biases for t;   a row with a mask:  v = -inf where t is not allowed, whatever it was (NaN too)
// Float32 throughout.  The bits say where counts have to be read at all: a vocabulary of 128,256 has 16 KB of them where the
// counts are 513 KB, so what a row reads beside its logits is 1/32 of them and a sector for every token it has said.
//
// Measured (device): 64 tokens appended 1.9 us, a launch and three dependent loads; 64 slots of 128,256 cleared 6.6 us (5.3 TB/s of
// stores) and 196,000 tokens added to them 4.9 us; 64 rows of 128,256 logits adjusted 17.9 us with 8,000 tokens seen, 100 biases and
// a mask on every second row, 11.5 as a copy (5.7 TB/s).  Biases alone, in place: 64 rows with 100 each 6.6 us, with 1,000 23.4, one row
// that names every token 0.51 ms (with a search through the row's list for each of its biases 11.1, 179 and 119 ms).
#include "common.cuh"
#include <initializer_list>

namespace {

constexpr int HT = 256, COARSE = 1024;

// ------------------------------------------------------------------- history
// 16 bytes a thread and step; a slot's row may start anywhere, so its ends are single words
__device__ __forceinline__ void clear(int* p, int n, int i, int step) {
  const int head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) / 4), quads = (n - head) / 4;
  if (i < head) p[i] = 0;
  for (int q = i; q < quads; q += step) reinterpret_cast<int4*>(p + head)[q] = make_int4(0, 0, 0, 0);
  const int tail = head + 4 * quads;
  if (i < n - tail) p[tail + i] = 0;
}
__global__ void __launch_bounds__(HT) history_reset_kernel(int* __restrict__ counts, int* __restrict__ seen,
                                                           const int* __restrict__ slots, int n_slots, int vocab, int words) {
  pdl_trigger();
  pdl_wait();
  const int slot = slots[blockIdx.y];
  if (slot < 0 || slot >= n_slots) return;
  const int i = blockIdx.x * HT + threadIdx.x, step = gridDim.x * HT;
  clear(counts + (size_t)slot * vocab, vocab, i, step);
  clear(seen + (size_t)slot * words, words, i, step);
}

// tokens[starts[r] .. starts[r + 1]) belong to slots[r]; the first n_prompt[r] of them are its prompt's.  starts null: token r.
__global__ void __launch_bounds__(HT) history_append_kernel(int* __restrict__ counts, int* __restrict__ seen,
                                                            const int* __restrict__ tokens, const int* __restrict__ slots,
                                                            const int* __restrict__ starts, const int* __restrict__ n_prompt,
                                                            int n_tokens, int n_requests, int n_slots, int vocab, int words) {
  __shared__ int coarse[COARSE];                       // every `stride`-th start: a search through memory is a chain of loads
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * HT + threadIdx.x;
  const int token = i < n_tokens ? tokens[i] : -1;     // under way during the search
  const int stride = (n_requests + COARSE - 1) / COARSE, n_coarse = (n_requests + stride - 1) / stride;
  if (starts != nullptr)
    for (int j = threadIdx.x; j < n_coarse; j += HT) coarse[j] = starts[j * stride];
  __syncthreads();
  int slot = -1, t = -1;
  bool generated = false;
  if (i < n_tokens) {
    int r = i, first = i, end = i + 1;
    if (starts != nullptr) {
      int lo = 0, hi = n_coarse;                       // the last request that starts at or before i
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (coarse[mid] <= i) lo = mid; else hi = mid;
      }
      lo *= stride;
      hi = min(n_requests, lo + stride);
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i) lo = mid; else hi = mid;
      }
      r = lo;
      first = starts[r];
      end = starts[r + 1];
    }
    if (i >= first && i < end) {
      slot = slots[r];
      t = token;
      generated = n_prompt == nullptr || i - first >= n_prompt[r];
    }
  }
  const bool ok = slot >= 0 && slot < n_slots && t >= 0 && t < vocab;
  if (ok && generated) atomicAdd(counts + (size_t)slot * vocab + t, 1);
  if (ok) atomicOr(seen + (size_t)slot * words + (t >> 5), (int)(1u << (t & 31)));
}

// -------------------------------------------------------------------- logits
struct AdjustParams {
  const void* logits;
  float* out;
  const int* slots;          // null: no penalties
  const float* penalties;    // [rows, 3]: r, p, f
  const int* counts;
  const int* seen;
  const int* bias_start;     // null: no biases
  const int* bias_ids;
  const float* bias_values;
  const int* mask_rows;      // null: no masks
  const int* masks;
  long long ld_in, ld_out;
  int vocab, words, n_slots, n_bias, n_masks, chunk, in_place;
};

// A block takes ADJUST_TOKENS (or fewer) logits of a row, in two passes.  The first copies them, -inf where the mask says so, V
// neighbours a thread (4 where all rows start on a whole vector, else 1) and ADJUST_STEPS of those under way at once; a thread whose
// tokens are all masked reads no logits.  The second goes over the tokens that have been seen, which the block lists first, one a
// thread: with some 4 in 100 of a vocabulary seen nearly every warp holds one, and the penalties' arithmetic on every logit takes
// longer than the memory does (64 rows of 128,256: 23 us against 12 so).  In place the first pass writes what is masked and no more.
constexpr int ADJUST_STEPS = 4, ADJUST_TOKENS = 4096;

// The biases of a block's tokens.  Every warp goes through the row's list and adds up those of an eighth of the tokens, in the list's order:
// the time is in proportion to the list, whatever it names and how often.  A sum that has not been begun is known by its bit in `named`
// (ADJUST_TOKENS of both).  Row, stretch and pointers are found again from the block's index, which passes for unknown: kept from the
// passes before they cost those registers (spills, 1.4 us).
__device__ __forceinline__ void add_biases(const AdjustParams& p, float* sums, unsigned* named) {
  int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  asm volatile("" : "+r"(row), "+r"(chunk), "+r"(tid));
  const int b0 = max(0, p.bias_start[row]), b1 = min(p.n_bias, p.bias_start[row + 1]);
  const int lo = chunk * p.chunk, hi = min(p.vocab, lo + p.chunk);
  const int mask_row = p.mask_rows != nullptr ? p.mask_rows[row] : -1;
  const int* mask = mask_row >= 0 && mask_row < p.n_masks ? p.masks + (size_t)mask_row * p.words : nullptr;
  const int* ids = p.bias_ids;
  const float* values = p.bias_values;
  float* out = p.out + row * p.ld_out;
  const auto takes = [&](int t) { return t >= lo && t < hi && !(mask && !((mask[t >> 5] >> (t & 31)) & 1)); };
  bool here = false;
  for (int j = b0 + tid; j < b1; j += HT) here |= takes(ids[j]);
  if (!__syncthreads_or(here)) return;                 // what was written before is there for the whole block
  const int lane = tid & 31, warp = tid >> 5;
  for (int j0 = b0 + lane; j0 - lane < b1; j0 += 32 * ADJUST_STEPS) {
    int next[ADJUST_STEPS];
#pragma unroll
    for (int s = 0; s < ADJUST_STEPS; ++s) next[s] = j0 + 32 * s < b1 ? ids[j0 + 32 * s] : -1;
#pragma unroll
    for (int s = 0; s < ADJUST_STEPS; ++s) {
      const int t = next[s], at = (int)((unsigned)t - (unsigned)lo);
      const bool mine = (t & 7) == warp && takes(t);
      const unsigned some = __ballot_sync(0xffffffffu, mine);
      if (some == 0) continue;
      if ((some & (some - 1)) == 0) {                  // one alone, as in a list that is short against the vocabulary
        if (mine) {
          const unsigned bit = 1u << (at & 31);
          sums[at] = ((named[at >> 5] & bit) ? sums[at] : 0.f) + values[j0 + 32 * s];
          atomicOr(&named[at >> 5], bit);
        }
        __syncwarp();
        continue;
      }
      const float v = mine ? values[j0 + 32 * s] : 0.f;
      const unsigned same = __match_any_sync(0xffffffffu, mine ? t : ~lane);     // lanes of the same token
      const bool first = mine && __ffs(same) - 1 == lane;
      float sum = first && ((named[at >> 5] >> (at & 31)) & 1) ? sums[at] : 0.f;
      for (unsigned left = some; left; left &= left - 1) {
        const int k = __ffs(left) - 1;
        const float vk = __shfl_sync(0xffffffffu, v, k);
        if ((same >> k) & 1) sum += vk;
      }
      if (first) {
        sums[at] = sum;
        atomicOr(&named[at >> 5], 1u << (at & 31));
      }
      __syncwarp();
    }
  }
  __syncthreads();
  static_assert(ADJUST_TOKENS / 16 == HT, "a thread has the bits of 16 tokens");
  for (unsigned bits = (named[tid >> 1] >> (16 * (tid & 1))) & 0xffffu; bits; bits &= bits - 1) {
    const int at = 16 * tid + __ffs(bits) - 1;
    out[lo + at] += sums[at];
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(HT, 8) adjust_logits_kernel(AdjustParams p) {
  __shared__ __align__(16) unsigned char shared[4 * ADJUST_TOKENS];
  unsigned short* list = reinterpret_cast<unsigned short*>(shared);    // tokens to penalise, from the block's first on, in no order that matters
  __shared__ unsigned named[ADJUST_TOKENS / 32];       // tokens that have biases
  __shared__ int listed;
  pdl_trigger();
  const int row = blockIdx.y, lo = blockIdx.x * p.chunk, hi = min(p.vocab, lo + p.chunk);     // a chunk is whole words of bits
  if (threadIdx.x == 0) listed = 0;
  if (threadIdx.x < ADJUST_TOKENS / 32) named[threadIdx.x] = 0u;
  __syncthreads();
  pdl_wait();
  const T* x = (const T*)p.logits + row * p.ld_in;
  float* out = p.out + row * p.ld_out;
  int slot = p.slots != nullptr ? p.slots[row] : -1;
  if (slot >= p.n_slots) slot = -1;
  int mask_row = p.mask_rows != nullptr ? p.mask_rows[row] : -1;
  if (mask_row >= p.n_masks) mask_row = -1;
  const int* seen = slot >= 0 ? p.seen + (size_t)slot * p.words : nullptr;
  const int* counts = slot >= 0 ? p.counts + (size_t)slot * p.vocab : nullptr;
  const int* mask = mask_row >= 0 ? p.masks + (size_t)mask_row * p.words : nullptr;
  if (seen) {
    for (int w = (lo >> 5) + threadIdx.x; w < (hi + 31) >> 5; w += HT) {
      unsigned bits = (unsigned)seen[w] & (mask ? (unsigned)mask[w] : 0xffffffffu);
      if (hi - 32 * w < 32) bits &= (1u << (hi - 32 * w)) - 1u;
      int at = bits ? atomicAdd(&listed, __popc(bits)) : 0;
      for (; bits; bits &= bits - 1) {
        const int i = 32 * w + __ffs(bits) - 1;
        list[at++] = (unsigned short)(i - lo);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(counts + i));      // the second pass's one trip to memory
      }
    }
  }
  if (!p.in_place || mask) {
    for (int i0 = lo + threadIdx.x * V; i0 < hi; i0 += HT * V * ADJUST_STEPS) {
      unsigned may[ADJUST_STEPS];                      // bits of the V tokens
      float v[ADJUST_STEPS][V];
      constexpr unsigned ALL = (1u << V) - 1u;
#pragma unroll
      for (int s = 0; s < ADJUST_STEPS; ++s) {
        const int i = i0 + s * HT * V;
        may[s] = mask && i < hi ? ((unsigned)mask[i >> 5] >> (i & 31)) & ALL : ALL;
      }
#pragma unroll
      for (int s = 0; s < ADJUST_STEPS; ++s) {
        const int i = i0 + s * HT * V;
        if (i < hi && may[s] && !(p.in_place && may[s] == ALL)) {
          if constexpr (V == 1) {
            v[s][0] = to_f32(x[i]);
          } else if constexpr (sizeof(T) == 4) {
            const float4 q = *reinterpret_cast<const float4*>(x + i);
            v[s][0] = q.x; v[s][1] = q.y; v[s][2] = q.z; v[s][3] = q.w;
          } else {
            const uint2 q = *reinterpret_cast<const uint2*>(x + i);
            v[s][0] = __uint_as_float(q.x << 16); v[s][1] = __uint_as_float(q.x & 0xffff0000u);
            v[s][2] = __uint_as_float(q.y << 16); v[s][3] = __uint_as_float(q.y & 0xffff0000u);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < ADJUST_STEPS; ++s) {
        const int i = i0 + s * HT * V;
        if (i >= hi || (p.in_place && may[s] == ALL)) continue;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (!((may[s] >> j) & 1)) v[s][j] = -INFINITY;
        if constexpr (V == 4) *reinterpret_cast<float4*>(out + i) = make_float4(v[s][0], v[s][1], v[s][2], v[s][3]);
        else out[i] = v[s][0];
      }
    }
  }
  if (seen) {
    __syncthreads();                                   // the list is whole, and the first pass's writes come before the second's
    const float factor = p.penalties[3 * row], once = p.penalties[3 * row + 1], each = p.penalties[3 * row + 2];
    for (int j = threadIdx.x; j < listed; j += HT) {
      const int t = lo + list[j], c = counts[t];
      float v = to_f32(x[t]);                          // in place: nobody has changed it, the mask lets it through
      v = v < 0.f ? v * factor : v / factor;
      if (c > 0) v -= each * (float)c + once;
      out[t] = v;
    }
  }
  if (p.bias_start == nullptr) return;
  add_biases(p, reinterpret_cast<float*>(shared), named);
}

}  // namespace

static int history_reset(int* counts, int* seen, const int* slots, int n, int n_slots, int vocab, cudaStream_t stream) {
  if (n <= 0 || vocab <= 0 || n_slots <= 0) return IE_OK;
  if (n > 65535) return IE_BAD_SIZE;
  const int blocks = (vocab + 32 * HT - 1) / (32 * HT);       // eight stores of 16 bytes a thread
  return launch_k(history_reset_kernel, dim3(blocks, n), HT, 0, stream, counts, seen, slots, n_slots, vocab, (vocab + 31) / 32);
}

static int history_append(int* counts, int* seen, const int* tokens, const int* slots, const int* starts, const int* n_prompt,
                          int n_tokens, int n_requests, int n_slots, int vocab, cudaStream_t stream) {
  if (n_tokens <= 0 || n_requests <= 0 || vocab <= 0 || n_slots <= 0) return IE_OK;
  if (starts == nullptr && n_tokens != n_requests) return IE_BAD_SIZE;
  return launch_k(history_append_kernel, (n_tokens + HT - 1) / HT, HT, 0, stream, counts, seen, tokens, slots, starts, n_prompt,
                  n_tokens, n_requests, n_slots, vocab, (vocab + 31) / 32);
}

static int adjust_logits(const void* logits, int dtype, float* out, const int* slots, const float* penalties, const int* counts,
                         const int* seen, const int* bias_start, const int* bias_ids, const float* bias_values,
                         const int* mask_rows, const int* masks, int n_rows, int vocab, long long ld_in, long long ld_out,
                         int n_slots, int n_bias, int n_masks, int in_place, cudaStream_t stream) {
  if (n_rows <= 0 || vocab <= 0) return IE_OK;
  if (n_rows > 65535) return IE_BAD_SIZE;
  if (dtype != IE_F32 && dtype != IE_BF16) return IE_BAD_DTYPE;
  AdjustParams p;
  p.logits = logits; p.out = out; p.slots = slots; p.penalties = penalties; p.counts = counts; p.seen = seen;
  p.bias_start = bias_start; p.bias_ids = bias_ids; p.bias_values = bias_values; p.mask_rows = mask_rows; p.masks = masks;
  p.ld_in = ld_in; p.ld_out = ld_out; p.vocab = vocab; p.words = (vocab + 31) / 32;
  p.n_slots = n_slots; p.n_bias = n_bias; p.n_masks = n_masks; p.in_place = in_place;
  const int size = dtype == IE_F32 ? 4 : 2;
  const bool vec = vocab % 4 == 0 && ((uintptr_t)logits & (4 * size - 1)) == 0 && ((uintptr_t)out & 15) == 0 &&
                   (n_rows == 1 || (ld_in % 4 == 0 && ld_out % 4 == 0));
  // 4,096 logits a block, or fewer where that would leave SMs without one
  const int sms = device_sms();
  if (sms <= 0) return IE_BAD_SIZE;
  p.chunk = ADJUST_TOKENS;
  while (p.chunk > 1024 && (long long)n_rows * ((vocab + p.chunk - 1) / p.chunk) < 2 * sms) p.chunk /= 2;
  const dim3 grid((vocab + p.chunk - 1) / p.chunk, n_rows);
  if (dtype == IE_F32)
    return vec ? launch_k(adjust_logits_kernel<float, 4>, grid, HT, 0, stream, p) : launch_k(adjust_logits_kernel<float, 1>, grid, HT, 0, stream, p);
  return vec ? launch_k(adjust_logits_kernel<bf16, 4>, grid, HT, 0, stream, p) : launch_k(adjust_logits_kernel<bf16, 1>, grid, HT, 0, stream, p);
}

// vectors and tables of words (of the logits: rows of them) that a call reads, or writes
static Span words(long long at, long long n) { return {(uintptr_t)at, 1, 4 * n, 4 * n}; }
static bool any_overlap(const Span& written, std::initializer_list<Span> others) {
  for (const Span& o : others)
    if (overlap(written, o)) return true;
  return false;
}

// the entries: arguments as 64-bit words in the order above, which a caller converts in one go; sizes above SIZE_MOST are refused
extern "C" int ie_history_reset(const long long* a) {
  if (beyond(a[3], a[4], a[5])) return IE_BAD_SIZE;
  const Span counts = words(a[0], a[4] * a[5]), seen = words(a[1], a[4] * ((a[5] + 31) / 32)), slots = words(a[2], a[3]);
  if (any_overlap(counts, {seen, slots}) || overlap(seen, slots)) return IE_OVERLAP;
  return history_reset((int*)a[0], (int*)a[1], (const int*)a[2], (int)a[3], (int)a[4], (int)a[5], (cudaStream_t)a[6]);
}
extern "C" int ie_history_append(const long long* a) {
  if (beyond(a[6], a[7], a[8], a[9])) return IE_BAD_SIZE;
  const Span counts = words(a[0], a[8] * a[9]), seen = words(a[1], a[8] * ((a[9] + 31) / 32));
  const Span tokens = words(a[2], a[6]), slots = words(a[3], a[7]), starts = words(a[4], a[7] + 1), n_prompt = words(a[5], a[7]);
  if (any_overlap(counts, {seen, tokens, slots, starts, n_prompt}) || any_overlap(seen, {tokens, slots, starts, n_prompt})) return IE_OVERLAP;
  return history_append((int*)a[0], (int*)a[1], (const int*)a[2], (const int*)a[3], (const int*)a[4], (const int*)a[5], (int)a[6],
                        (int)a[7], (int)a[8], (int)a[9], (cudaStream_t)a[10]);
}
extern "C" int ie_adjust_logits(const long long* a) {
  if (beyond(a[12], a[13], a[16], a[17], a[18])) return IE_BAD_SIZE;
  const long long rows = a[12], vocab = a[13], bits = (vocab + 31) / 32;      // out against logits is the caller's, who knows whether they are one
  const Span out = {(uintptr_t)a[2], rows, 4 * vocab, 4 * a[15]};
  if (any_overlap(out, {words(a[3], rows), words(a[4], 3 * rows), words(a[5], a[16] * vocab), words(a[6], a[16] * bits), words(a[7], rows + 1),
                        words(a[8], a[17]), words(a[9], a[17]), words(a[10], rows), words(a[11], a[18] * bits)})) return IE_OVERLAP;
  return adjust_logits((const void*)a[0], (int)a[1], (float*)a[2], (const int*)a[3], (const float*)a[4], (const int*)a[5],
                       (const int*)a[6], (const int*)a[7], (const int*)a[8], (const float*)a[9], (const int*)a[10], (const int*)a[11],
                       (int)a[12], (int)a[13], a[14], a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19], (cudaStream_t)a[20]);
}
