// Choice of one token per row of 32-bit logits with temperature, top-k, top-p and min-p, from uniform numbers that the caller gives.
//
// A row's tokens are ordered by logit, larger first, the lower id first among equals (NaN last).  With m the largest logit and T the
// temperature, token i weighs w_i = exp((l_i - m) / T).  Kept is the shortest of three prefixes of that order: top_k tokens (top_k <= 0:
// all); the fewest whose weights reach top_p of the weight that top_k leaves (top_p >= 1: all); those with w_i >= min_p; and the first
// token always.  Drawn is the first kept token, in order of ids, at which the running sum of kept weights exceeds u times their sum.
// Rows with T <= 0, and rows whose largest logit is not above -infinity, give the first token of the order.  A logit of +infinity leaves weight to such logits alone.
//
// Weights are whole numbers of 2^-44: their sums are exact in 64 bits (2^19 tokens at most), so that no sum depends on the order it is
// taken in, on how a row is spread over threads and blocks, or on which atomic came first.  What is left of rounding is a weight's own error, a few 2^-25 of
// it: with sums in 32-bit floats the border of top-p, and the token that a number falls on, would be off by a token in one draw of some hundred over a flat row.
#include "common.cuh"

namespace tlie {

constexpr int kFilterThreads = 1024;
constexpr int kFilterMaxVocab = 1 << 19;
constexpr int kWeightBits = 44;

// Logits as unsigned numbers of the same order: equal floats are equal numbers (-0 counts as 0), NaN is below everything.
__device__ __forceinline__ unsigned logit_key(float l) {
  if (l != l) return 0u;
  const int bits = __float_as_int(l + 0.0f);
  return bits < 0 ? ~(unsigned)bits : (unsigned)bits | 0x80000000u;
}

// log2(e) / T in two floats.  Temperatures below 1e-30 count as 1e-30: to differ there two logits would have to lie 1e-29 apart.
struct Scale {
  float high, low;
};
__device__ __forceinline__ Scale weight_scale(float temperature) {
  const double c = 1.4426950408889634074 / (double)fmaxf(temperature, 1e-30f);
  Scale s;
  s.high = (float)c;
  s.low = (float)(c - (double)s.high);
  return s;
}

// exp((l - m) / T) in units of 2^-44.  The exponent's difference and product are kept in two floats (what rounding takes off one is in the other), so that
// its error does not grow with the distance from m.  2^f on [-1/2, 1/2] is a polynomial of degree 6 (least maximum of the relative error, 2e-9).
__device__ __forceinline__ unsigned long long token_weight(float l, float m, Scale c) {
  if (l == m) return 1ull << kWeightBits;
  const float s = l - m, back = s - l;
  const float e = (l - (s - back)) - (m + back);
  const float high = s * c.high;
  if (!(high >= -46.0f)) return 0ull;   // (NaN and infinities too)
  const float low = fmaf(s, c.high, -high) + fmaf(s, c.low, e * c.high);
  const float rounded = high + 12582912.0f;   // 1.5 * 2^23: the whole number nearest to it in the lower bits
  const int n = __float_as_int(rounded) - 0x4B400000;
  const float f = (high - (rounded - 12582912.0f)) + low;
  float p = 1.5353153867181391e-4f;
  p = fmaf(p, f, 1.339913229458034e-3f);
  p = fmaf(p, f, 9.618439711630344e-3f);
  p = fmaf(p, f, 5.550331994891167e-2f);
  p = fmaf(p, f, 2.4022647738456726e-1f);
  p = fmaf(p, f, 6.931471824645996e-1f);
  p = fmaf(p, f, 1.0f);
  const unsigned bits = __float_as_uint(p);
  const int down = 127 - (int)(bits >> 23) - n;   // 0 to 47: how far below 1 the leading bit lies
  const unsigned long long mantissa = (unsigned long long)((bits & 0x7fffffu) | 0x800000u) << (kWeightBits - 23);
  return mantissa >> down;
}

__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long* scratch /* >= 32 */) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x % 32 < blockDim.x / 32 ? scratch[threadIdx.x & 31] : 0ull;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}

// The last token of a prefix of the order: tokens with a larger key, and those of this key up to this id, belong to it.
struct Border {
  unsigned key;
  int id;
  __device__ bool holds(unsigned k, int i) const { return k > key || (k == key && i <= id); }
  __device__ bool before(const Border& o) const { return o.holds(key, id); }   // no longer than o's prefix
};

// One block per row.  A border is found by bisecting first on the key, then, among tokens of that key, on the id.
__global__ void __launch_bounds__(kFilterThreads)
    sample_filtered_kernel(const float* __restrict__ logits, long long row_stride, int all_rows, int vocab, const int* __restrict__ rows, const float* __restrict__ temperature,
                           const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniforms,
                           int* __restrict__ out) {
  __shared__ unsigned long long scratch[32];
  __shared__ unsigned long long prefix[kFilterThreads];
  __shared__ unsigned long long best;
  __shared__ int chosen;
  const int index = rows != nullptr ? rows[blockIdx.x] : (int)blockIdx.x;
  if (index < 0 || index >= all_rows) return;
  const float* row = logits + (size_t)index * row_stride;

  if (threadIdx.x == 0) best = 0ull;
  __syncthreads();
  unsigned long long mine = 0ull;   // key, then the id's complement: the larger of two is the earlier in the order
  for (int i = threadIdx.x; i < vocab; i += blockDim.x) mine = max(mine, ((unsigned long long)logit_key(row[i]) << 32) | (unsigned)~i);
  atomicMax(&best, mine);
  __syncthreads();
  const int first = (int)~(unsigned)best;
  const float m = row[first];
  const float temp = temperature[blockIdx.x];
  if (!(temp > 0.0f) || !(m > -INFINITY)) {
    if (threadIdx.x == 0) out[index] = m == m ? first : 0;   // a row of NaN: token 0
    return;
  }
  const Scale scale = weight_scale(temp);
  const Border all = {0u, vocab};

  // What the tokens of `within` bring that `border` holds: their number or their weight.
  auto measure = [&](const Border& within, const Border& border, bool weights) {
    unsigned long long sum = 0ull;
    for (int i = threadIdx.x; i < vocab; i += blockDim.x) {
      const float l = row[i];
      const unsigned k = logit_key(l);
      if (within.holds(k, i) && border.holds(k, i)) sum += weights ? token_weight(l, m, scale) : 1ull;
    }
    return block_sum_u64(sum, scratch);
  };
  // The shortest prefix of the order that brings `wanted` (which all of `within` does).
  auto find = [&](const Border& within, unsigned long long wanted, bool weights) {
    unsigned low = 0u, high = 0xffffffffu;   // the tokens with key >= low bring it, those with key >= high (NaN has no such key) do not
    while (high - low > 1u) {
      const unsigned middle = low + (high - low) / 2u;
      if (measure(within, {middle, vocab}, weights) >= wanted) low = middle;
      else high = middle;
    }
    int none = -1, enough = vocab;
    while (enough - none > 1) {
      const int middle = none + (enough - none) / 2;
      if (measure(within, {low, middle}, weights) >= wanted) enough = middle;
      else none = middle;
    }
    return Border{low, enough};
  };

  Border kept = all;
  const int k = top_k[blockIdx.x];
  if (k > 0 && k < vocab) kept = find(all, (unsigned long long)k, false);
  const float p = top_p[blockIdx.x];
  const float smallest = min_p[blockIdx.x];
  unsigned long long floor_weight = 0ull;
  if (smallest > 0.0f) floor_weight = smallest >= 1.0f ? 1ull << kWeightBits : (unsigned long long)ceil((double)smallest * (double)(1ull << kWeightBits));
  if (p < 1.0f) {
    const unsigned long long total = measure(all, kept, true);
    const unsigned long long wanted = p > 0.0f ? (unsigned long long)ceil((double)p * (double)total) : 1ull;
    kept = find(kept, max(1ull, min(wanted, total)), true);
  }
  const bool first_only = smallest > 1.0f;
  auto weight = [&](int i) -> unsigned long long {
    const float l = row[i];
    if (!kept.holds(logit_key(l), i) || (first_only && i != first)) return 0ull;
    const unsigned long long w = token_weight(l, m, scale);
    return w >= floor_weight ? w : 0ull;
  };

  // consecutive tokens per thread, so that the walk is in order of ids
  const int each = (vocab + blockDim.x - 1) / blockDim.x;
  const int begin = min(vocab, (int)threadIdx.x * each), end = min(vocab, begin + each);
  unsigned long long sum = 0ull;
  for (int i = begin; i < end; ++i) sum += weight(i);
  const unsigned long long total = block_sum_u64(sum, scratch);
  prefix[threadIdx.x] = sum;
  __syncthreads();
  unsigned long long start = 0ull;
  for (int t = 0; t < (int)threadIdx.x; ++t) start += prefix[t];
  const float u = uniforms[blockIdx.x];
  unsigned long long target = u > 0.0f ? (unsigned long long)((double)fminf(u, 1.0f) * (double)total) : 0ull;
  if (target >= total) target = total - 1ull;
  if (threadIdx.x == 0) chosen = first;
  __syncthreads();
  if (target >= start && target < start + sum) {
    int i = begin;
    for (unsigned long long running = start + weight(i); running <= target; running += weight(i)) ++i;
    chosen = i;
  }
  __syncthreads();
  if (threadIdx.x == 0) out[index] = chosen;
}

__global__ void uniforms_kernel(const long long* __restrict__ seeds, const long long* __restrict__ counters, float* __restrict__ out, int count) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= count) return;
  // splitmix64's finaliser over (seed, counter), 24 bits of it: the uniform number of a request's draw, as the other sampling kernels make it
  unsigned long long z = (unsigned long long)seeds[i] * 0x9E3779B97F4A7C15ull + ((unsigned long long)counters[i] + 1ull) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z = z ^ (z >> 31);
  out[i] = (float)(z >> 40) * (1.0f / 16777216.0f);
}

}  // namespace tlie

using namespace tlie;

// logits: all_rows rows of vocab, row_stride elements apart.  rows (or null: row r for all r): which of them the r-th option set is for; numbers outside
// [0, all_rows) are passed over.  out: one token per row of the logits.
TLIE_EXPORT int tlie_sample_filtered(const float* logits, long long row_stride, int all_rows, int vocab, const int* rows, int count, const float* temperature,
                                     const int* top_k, const float* top_p, const float* min_p, const float* uniforms, int* out, cudaStream_t stream) {
  if (count <= 0) return 0;
  if (vocab <= 0 || vocab > kFilterMaxVocab || row_stride < 0) return (int)cudaErrorInvalidValue;
  sample_filtered_kernel<<<count, kFilterThreads, 0, stream>>>(logits, row_stride, all_rows, vocab, rows, temperature, top_k, top_p, min_p, uniforms, out);
  return (int)cudaGetLastError();
}

TLIE_EXPORT int tlie_uniforms(const long long* seeds, const long long* counters, float* out, int count, cudaStream_t stream) {
  if (count <= 0) return 0;
  uniforms_kernel<<<(count + 255) / 256, 256, 0, stream>>>(seeds, counters, out, count);
  return (int)cudaGetLastError();
}
