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
#include "common.cuh"

namespace {

constexpr int HT = 256;

// ------------------------------------------------------------------- history
__global__ void __launch_bounds__(HT) history_reset_kernel(int* __restrict__ counts, int* __restrict__ seen,
                                                           const int* __restrict__ slots, int n_slots, int vocab, int words) {
  pdl_trigger();
  pdl_wait();
  const int slot = slots[blockIdx.y];
  if (slot < 0 || slot >= n_slots) return;
  int* c = counts + (size_t)slot * vocab;
  int* s = seen + (size_t)slot * words;
  for (int i = blockIdx.x * HT + threadIdx.x; i < vocab; i += gridDim.x * HT) c[i] = 0;
  for (int i = blockIdx.x * HT + threadIdx.x; i < words; i += gridDim.x * HT) s[i] = 0;
}

// tokens[starts[r] .. starts[r + 1]) belong to slots[r]; the first n_prompt[r] of them are its prompt's.  starts null: token r.
__global__ void __launch_bounds__(HT) history_append_kernel(int* __restrict__ counts, int* __restrict__ seen,
                                                            const int* __restrict__ tokens, const int* __restrict__ slots,
                                                            const int* __restrict__ starts, const int* __restrict__ n_prompt,
                                                            int n_tokens, int n_requests, int n_slots, int vocab, int words) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * HT + threadIdx.x;
  if (i >= n_tokens) return;
  int r = i, first = i;
  if (starts != nullptr) {
    int lo = 0, hi = n_requests;                     // the last request that starts at or before i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= i) lo = mid; else hi = mid;
    }
    r = lo;
    first = starts[r];
    if (i < first || i >= starts[r + 1]) return;
  }
  const int slot = slots[r], t = tokens[i];
  if (slot < 0 || slot >= n_slots || t < 0 || t >= vocab) return;
  if (n_prompt == nullptr || i - first >= n_prompt[r]) atomicAdd(counts + (size_t)slot * vocab + t, 1);
  atomicOr(seen + (size_t)slot * words + (t >> 5), (int)(1u << (t & 31)));
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

template <typename T>
__global__ void __launch_bounds__(HT) adjust_logits_kernel(AdjustParams p) {
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y, lo = blockIdx.x * p.chunk, hi = min(p.vocab, lo + p.chunk);
  const T* x = (const T*)p.logits + row * p.ld_in;
  float* out = p.out + row * p.ld_out;
  int slot = p.slots != nullptr ? p.slots[row] : -1;
  if (slot >= p.n_slots) slot = -1;
  int mask_row = p.mask_rows != nullptr ? p.mask_rows[row] : -1;
  if (mask_row >= p.n_masks) mask_row = -1;
  const int* seen = slot >= 0 ? p.seen + (size_t)slot * p.words : nullptr;
  const int* counts = slot >= 0 ? p.counts + (size_t)slot * p.vocab : nullptr;
  const int* mask = mask_row >= 0 ? p.masks + (size_t)mask_row * p.words : nullptr;
  float factor = 1.f, once = 0.f, each = 0.f;
  if (seen) { factor = p.penalties[3 * row]; once = p.penalties[3 * row + 1]; each = p.penalties[3 * row + 2]; }
  for (int i = lo + threadIdx.x; i < hi; i += HT) {
    float v = to_f32(x[i]);
    if (seen && (seen[i >> 5] >> (i & 31)) & 1) {
      v = v < 0.f ? v * factor : v / factor;
      const int c = counts[i];
      if (c > 0) v -= each * (float)c + once;
    }
    if (mask && !((mask[i >> 5] >> (i & 31)) & 1)) v = -INFINITY;
    out[i] = v;
  }
  if (p.bias_start == nullptr) return;
  const int b0 = max(0, p.bias_start[row]), b1 = min(p.n_bias, p.bias_start[row + 1]);
  if (b0 >= b1) return;
  __syncthreads();
  for (int b = b0 + threadIdx.x; b < b1; b += HT) {
    const int t = p.bias_ids[b];
    if (t < lo || t >= hi || (mask && !((mask[t >> 5] >> (t & 31)) & 1))) continue;
    bool first = true;
    for (int j = b0; j < b && first; ++j) first = p.bias_ids[j] != t;
    if (!first) continue;
    float sum = p.bias_values[b];                    // a token that comes twice: its biases in order, by one thread
    for (int j = b + 1; j < b1; ++j)
      if (p.bias_ids[j] == t) sum += p.bias_values[j];
    out[t] += sum;
  }
}

}  // namespace

extern "C" int ie_history_reset(int* counts, int* seen, const int* slots, int n, int n_slots, int vocab, cudaStream_t stream) {
  if (n <= 0 || vocab <= 0 || n_slots <= 0) return IE_OK;
  if (n > 65535) return IE_BAD_SIZE;
  const int blocks = (vocab + 4 * HT - 1) / (4 * HT);
  return launch_k(history_reset_kernel, dim3(blocks, n), HT, 0, stream, counts, seen, slots, n_slots, vocab, (vocab + 31) / 32);
}

extern "C" int ie_history_append(int* counts, int* seen, const int* tokens, const int* slots, const int* starts, const int* n_prompt,
                                 int n_tokens, int n_requests, int n_slots, int vocab, cudaStream_t stream) {
  if (n_tokens <= 0 || n_requests <= 0 || vocab <= 0 || n_slots <= 0) return IE_OK;
  if (starts == nullptr && n_tokens != n_requests) return IE_BAD_SIZE;
  return launch_k(history_append_kernel, (n_tokens + HT - 1) / HT, HT, 0, stream, counts, seen, tokens, slots, starts, n_prompt,
                  n_tokens, n_requests, n_slots, vocab, (vocab + 31) / 32);
}

extern "C" int ie_adjust_logits(const void* logits, int dtype, float* out, const int* slots, const float* penalties, const int* counts,
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
  p.n_slots = n_slots; p.n_bias = n_bias; p.n_masks = n_masks; p.chunk = 4096; p.in_place = in_place;
  const dim3 grid((vocab + p.chunk - 1) / p.chunk, n_rows);
  return dtype == IE_F32 ? launch_k(adjust_logits_kernel<float>, grid, HT, 0, stream, p)
                         : launch_k(adjust_logits_kernel<bf16>, grid, HT, 0, stream, p);
}
