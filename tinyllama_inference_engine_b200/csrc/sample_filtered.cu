// Choice of one token per row of 32-bit logits with temperature, top-k, top-p and min-p, from uniform numbers that the caller gives.
//
// A row's tokens are ordered by logit, larger first, the lower id first among equals (NaN last).  With m the largest logit and T the
// temperature, token i weighs w_i = exp((l_i - m) / T).  Kept is the shortest of three prefixes of that order: top_k tokens (top_k <= 0:
// all); the fewest whose weights reach top_p of the weight that top_k leaves (top_p >= 1: all); those with w_i >= min_p; and the first
// token always.  Drawn is the first kept token, in order of ids, at which the running sum of kept weights exceeds u times their sum.
// Rows with T <= 0, and rows whose largest logit is not above -infinity, give the first token of the order.  A logit of +infinity leaves weight to such logits alone.
//
// Weights are whole numbers of 2^-44: their sums are exact in 64 bits, so that no sum depends on the order it is
// taken in, on how a row is spread over threads and blocks, or on which atomic came first.  What is left of rounding is a weight's own error, a few 2^-25 of
// it: with sums in 32-bit floats the border of top-p, and the token that a number falls on, would be off by a token in one draw of some hundred over a flat row.
#include <cooperative_groups.h>

#include <cstdlib>

#include "common.cuh"

namespace tlie {

constexpr int kFilterThreads = 512, kFilterWarps = kFilterThreads / 32;
constexpr int kBinBits = 11, kBins = 1 << kBinBits, kBinsEach = kBins / kFilterThreads;
constexpr int kListed = kFilterThreads;    // tokens of the list, one per thread
constexpr int kEarly = 3 * kFilterThreads; // ... and of those that may come on it, while a row is read
constexpr int kFilterMaxVocab = 1 << 19;   // (so many weights of 2^44 and less: sums fit 64 bits, a token's id and weight one number)
constexpr int kWeightBits = 44;

// Logits as unsigned numbers of the same order: equal floats are equal numbers (-0 counts as 0), NaN is below everything.
__device__ __forceinline__ unsigned logit_key(float l) {
  if (l != l) return 0u;
  const int bits = __float_as_int(l + 0.0f);
  return bits < 0 ? ~(unsigned)bits : (unsigned)bits | 0x80000000u;
}

// What a row's weights are made with: y = l c - m c in 64 bits is log2 of one, with c = log2(e) / T.  Temperatures outside 1e-30 to 1e30 count as the nearer of these: to
// differ below two logits would have to lie 1e-29 apart, and above nothing differs.
struct Scale {
  double c, mc;
};
__device__ __forceinline__ Scale weight_scale(float temperature, float m) {
  const double c = 1.4426950408889634074 / (double)fminf(fmaxf(temperature, 1e-30f), 1e30f);
  return Scale{c, (double)m * c};
}

// exp((l - m) / T) in units of 2^-44.  y with 23 bits behind the point stands in the lower word of y + 1.5 * 2^29, its whole part (rounded down) and the rest f, put behind a
// 1, are what a float of 1 + f is made of.  2^(f - 1/2) sqrt(2) is a polynomial of degree 6 in f - 1/2 (least maximum of the relative error, 2e-8 with its coefficients rounded).
__device__ __forceinline__ unsigned long long token_weight(float l, float m, Scale c) {
  const double y = fma((double)l, c.c, -c.mc);
  const unsigned size = (unsigned)__double2hiint(y) ^ 0x80000000u;   // below that of 46 for -46 < y < 0; NaN, infinities and y >= 0 (the maximum itself) are above
  const int fixed = __double2loint(y + 805306368.0);
  const float f = __int_as_float((fixed & 0x7fffff) | 0x3f800000) - 1.5f;
  float p = 2.170223742723465e-4f;
  p = fmaf(p, f, 1.8950358498841524e-3f);
  p = fmaf(p, f, 1.3602597638964653e-2f);
  p = fmaf(p, f, 7.849350571632385e-2f);
  p = fmaf(p, f, 3.397315442562103e-1f);
  p = fmaf(p, f, 9.802581667900085e-1f);
  p = fmaf(p, f, 1.4142135381698608f);
  const unsigned bits = __float_as_uint(p);
  const int down = 127 - (int)(bits >> 23) - (fixed >> 23);   // 0 to 47: how far below 1 the leading bit lies
  const unsigned long long w = ((unsigned long long)((bits & 0x7fffffu) | 0x800000u) << (kWeightBits - 23)) >> down;
  return l == m ? 1ull << kWeightBits : size < 0x40470000u ? w : 0ull;
}

// The last token of a prefix of the order: tokens with a larger key, and those of this key up to this id, belong to it.
struct Border {
  unsigned key;
  int id;
  __device__ bool holds(unsigned k, int i) const { return k > key || (k == key && i <= id); }
};

// A row belongs to a cluster of CTAs, consecutive tokens to each, which read them once for the maximum and again, from the caches, for what follows; that is mostly done by the first CTA on a short
// list of the order's first tokens.  As many threads' maxima as are asked for bound the list from below (so many tokens at least are not below the least of them), and the highest
// of the CTAs' bounds holds for all.  With top_k so many tokens are asked for and all others are out of it; with top_p alone some hundred, and what all tokens weigh, to some 2^-19 of it, tells whether
// they suffice and where the border lies; only if it would lie elsewhere for another total in between are all weights worked out exactly (with exact weights at once, 21 instructions a token,
// 64 rows of 128,256 took 35.5 us).  min_p alone says itself which tokens it leaves.  One row is bound by the chain of its steps (32,000 tokens, top-k 40 and top-p: 10.7 us, top-p alone: 15.3);
// many by reading (256 rows of 128,256 with top-k 50: 39.7 us, 3.3 TB/s; reading ahead through shared memory took 2 more) and, with top-p alone, by the second pass and the slowest CTA of a
// cluster (64 rows of 128,256: 26.1 us).
//
// Where the list does not do (top_k beyond it, flat rows), a border is found from a histogram over 2,048 runs of logits, 1/64 wide, below the largest, of numbers or
// of exact weights, and from the tokens of the run that it falls in, which the first CTA sorts.  Where those are too many (equal logits, or very close ones) the run is
// cut by the bits of the logits, and equal ones by id.  (One row of 32,000 with top-k 450: 33 us, 47 with top-p 0.95 beside it; 160 rows of 128,256 with top-k 400: 313 and 435, with 300, on the list: 76 and 74; 64 rows at a
// temperature of 3 with top-p alone: 125.)
struct FilterShared {
  union {                         // (one is done with before the other begins)
    struct {
      unsigned low[kBins], high[kBins];   // a histogram's numbers, 64 bits in two words: an atomic of 64 bits on shared memory is a loop
    };
    unsigned long long list[kListed];
  };
  unsigned long long exchange[2][kFilterThreads], early[kEarly];
  unsigned long long scan[kFilterWarps];
  unsigned long long gather[2][2][8];   // two numbers per CTA
  unsigned long long above;       // the first CTA's are the cluster's, as are:
  unsigned long long wanted;
  int bin, listed, chosen, found_id;
  unsigned found_key;
  int last_run[2];
  unsigned least[2];
};

__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}
__device__ __forceinline__ unsigned long long warp_prefix_u64(unsigned long long v, int lane) {   // the sum up to and with this lane
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, v, offset);
    if (lane >= offset) v += other;
  }
  return v;
}
// Sum over the CTA's threads before this one, and of all.
__device__ __noinline__ unsigned long long block_prefix(unsigned long long v, unsigned long long* scan, unsigned long long& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long upto = warp_prefix_u64(v, lane);
  __syncthreads();
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  unsigned long long before = 0ull, sum = 0ull;
#pragma unroll
  for (int w = 0; w < kFilterWarps; ++w) {
    const unsigned long long here = scan[w];
    if (w < warp) before += here;
    sum += here;
  }
  all = sum;
  return before + upto - v;
}
// The first n threads' numbers (all different) in falling order, one per thread (n and more: whatever is there, below all others).  Most of what a sort takes is the fetching of
// code that no other warp has fetched before: loops are left as loops.
__device__ __noinline__ unsigned long long sort_falling(unsigned long long v, int n, unsigned long long (&exchange)[2][kFilterThreads]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();   // (a sort before may still be read)
  if (n <= 64) {     // few: a number's place is how many are above it, counted by eight threads side by side
    exchange[0][threadIdx.x] = v;
    __syncthreads();
    const int i = threadIdx.x / 8;
    const unsigned long long mine = i < n ? exchange[0][i] : 0ull;
    unsigned place = 0u;
    for (int j = threadIdx.x & 7; j < n; j += 8) place += exchange[0][j] > mine;
    for (int offset = 1; offset < 8; offset <<= 1) place += __shfl_xor_sync(0xffffffffu, place, offset);
    if (i < n && (threadIdx.x & 7) == 0) exchange[1][place] = mine;
    __syncthreads();
    return (int)threadIdx.x < n ? exchange[1][threadIdx.x] : 0ull;
  }
  // Every warp puts its 32 in order by exchanges; a number's place is its place there and how many of each other warp's are above it, found by halving.  (53 numbers by counting: 1,340 cycles;
  // 219 by halving: 6,200 beside another CTA's work.)
  if ((int)threadIdx.x >= n) v = 0ull;
  if (warp * 32 < n) {
#pragma unroll 1
    for (int run = 2; run <= 32; run *= 2)
#pragma unroll 1
      for (int reach = run / 2; reach > 0; reach /= 2) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, reach);
        const bool larger = ((lane & reach) == 0) == (run == 32 || (lane & run) == 0);
        if ((other > v) == larger) v = other;
      }
  }
  exchange[0][threadIdx.x] = v;
  __syncthreads();
  if (warp * 32 < n) {
    int place = lane;
    const int runs = (n + 31) / 32;
    for (int r = 0; r < runs; ++r) {
      const unsigned long long* in_order = exchange[0] + r * 32;
      int above = 0;
#pragma unroll
      for (int step = 16; step > 0; step /= 2) above += in_order[above + step - 1] > v ? step : 0;
      place += r != warp ? above + (in_order[above] > v ? 1 : 0) : 0;
    }
    if (lane < n - warp * 32) exchange[1][place] = v;
  }
  __syncthreads();
  return (int)threadIdx.x < n ? exchange[1][threadIdx.x] : 0ull;
}
__device__ __forceinline__ float key_logit(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// One row, by the threads of a cluster.
class RowFilter {
 public:
  __device__ RowFilter(FilterShared& shared, const float* row, int vocab, int slice)
      : sh(shared), cluster(cooperative_groups::this_cluster()), vocab(vocab), ctas(cluster.num_blocks()), rank(cluster.block_rank()),
        lane(threadIdx.x & 31), warp(threadIdx.x >> 5), first_id(min(vocab, rank * slice)), count(min(vocab, (rank + 1) * slice) - first_id), tokens(row + first_id),
        head(min(count, (int)((4 - (reinterpret_cast<uintptr_t>(row + first_id) >> 2 & 3)) & 3))), quads((count - head) >> 2) {}

  // The row's token, in the first CTA.
  __device__ int choose(float temperature, int top_k, float top_p, float min_p, float u) {
    const bool by_number = top_k > 0 && top_k < vocab, by_weight = top_p < 1.0f;
    const bool first_only = !(temperature > 0.0f) || top_k == 1 || min_p > 1.0f || top_p <= 0.0f;
    const int asked = first_only ? 0 : by_number ? top_k : by_weight ? kGuess : 0;
    const bool early = ctas == 1 && by_number && !first_only && top_k <= kFilterThreads;
    load(early ? asked : 0);
    const float largest = block_max(thread_max);   // this CTA's
    // What all of the tokens asked for are not below in one CTA, and what a CTA's share of them is not below in any.
    uint2 bounds = make_uint2(logit_key(-INFINITY), logit_key(-INFINITY));
    if (asked > 0 && largest > -INFINITY) bounds = least_of_maxima(largest, asked, (asked + ctas - 1) / ctas);
    arrived();
    const unsigned long long* all = gather(logit_key(largest), ((unsigned long long)bounds.x << 32) | bounds.y);
    unsigned key = 0u, in_one = 0u, in_any = 0xffffffffu;
    for (int c = 0; c < ctas; ++c) key = max(key, (unsigned)all[c]), in_one = max(in_one, (unsigned)(all[8 + c] >> 32)), in_any = min(in_any, (unsigned)all[8 + c]);
    m = key_logit(key);
    float bound = key_logit(max(in_one, in_any));
    if (!any_token(key)) return 0;                        // a row of NaN
    if (first_only || !(m > -INFINITY)) return first_of_order();

    scale = weight_scale(temperature, m);
    floor_weight = min_p > 0.0f ? (unsigned long long)ceil((double)min_p * (double)(1ull << kWeightBits)) : 0ull;
    if (early) {   // of the tokens listed on the way those that are not below the bound of all
      const int listed = sh.listed;
      __syncthreads();
      if (threadIdx.x == 0) sh.listed = 0;
      __syncthreads();
      if (listed >= top_k && listed <= kEarly) {
        for (int i = threadIdx.x; i < listed; i += kFilterThreads) {
          const unsigned long long token = sh.early[i];
          if ((unsigned)(token >> 32) < bounds.x) continue;
          const int at = atomicAdd(&sh.listed, 1);
          if (at < kListed) sh.list[at] = token;
        }
        __syncthreads();
        if (sh.listed <= kListed) return choose_from_list(top_k, top_p, 0ull, 0ull, u);
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
      }
    }
    const bool by_floor = !by_number && !by_weight && floor_weight > 0ull;
    if (by_floor) bound = m + temperature * (logf(min_p) * 1.0001f - 0.001f);   // (a little low: the list is longer than what stays of it)
    if (bound > -INFINITY) {
      const bool nucleus = by_weight && !by_number;
      unsigned long long mine = 0ull, least = 0ull, most = 0ull;
      float spread = 0.0f;
      list_from(bound, nucleus, mine, spread);
      if (nucleus) {   // between what two numbers the weight of all tokens lies
        mine = warp_sum_u64(mine);
        unsigned long long spread_of_all = warp_sum_u64(spread_in_units(spread));
        if (lane == 0) sh.scan[warp] = mine, sh.exchange[0][warp] = spread_of_all;
        __syncthreads();
        mine = spread_of_all = 0ull;
        for (int w = 0; w < kFilterWarps; ++w) mine += sh.scan[w], spread_of_all += sh.exchange[0][w];
        all = gather(mine, spread_of_all);
        unsigned long long total = 0ull, far = 0ull;
        for (int c = 0; c < ctas; ++c) total += all[c], far += all[8 + c];
        const unsigned long long off = off_at_most(total, far);
        least = total - min(total, off), most = total + off;
      } else {
        sync();
      }
      if (*at_first(&sh.listed) <= kListed) {
        if (by_number || by_floor) return rank == 0 ? choose_from_list(by_number ? top_k : kListed, top_p, 0ull, 0ull, u) : 0;
#pragma unroll 1
        for (int exact = m < INFINITY ? 0 : 1; exact < 2; ++exact) {
          if (exact) {
            mine = 0ull;
            for_tokens([&](float l, int) { mine += weight(l); });
            block_prefix(mine, sh.scan, mine);
            all = gather(mine, 0ull);
            least = 0ull;
            for (int c = 0; c < ctas; ++c) least += all[c];
            most = least;
          }
          if (rank == 0) {
            const int token = choose_from_list(kListed, top_p, least, most, u);
            if (threadIdx.x == 0) sh.chosen = token;
          }
          sync();
          const int token = *at_first(&sh.chosen);
          if (token >= 0) return token;
          if (token == kListTooShort) break;
        }
      }
      sync();   // (all have read the list's length before the next search clears it)
    }
    if (!by_number && !by_weight && floor_weight == 0ull) {   // all tokens
      const int token = m < INFINITY ? draw_from_all<false>(u) : -1;
      if (token >= 0) return token;
      sync();   // (all have read it)
      return draw_from_all<true>(u);
    }
    Border kept = {0u, vocab};
#pragma unroll 1
    for (int by = 0; by < 2; ++by)
      if (by == 0 ? by_number : by_weight) kept = find(kept, (unsigned long long)top_k, by == 1, top_p);
    return draw(kept, u);
  }

  __device__ void arrive() {   // (a CTA's shared memory may be written once the CTA runs)
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  }

 private:
  static constexpr int kGuess = 192, kListTooShort = -1, kUnsure = -2;
  FilterShared& sh;
  cooperative_groups::cluster_group cluster;
  const int vocab, ctas, rank, lane, warp, first_id, count;
  const float* tokens;     // this CTA's: `head` of them in front of the first 16 bytes, `quads` times four, and what is left
  const int head, quads;
  float m, thread_max;
  Scale scale;
  unsigned long long floor_weight;
  int gathers = 0;

  __device__ static bool any_token(unsigned key) { return key != 0u; }
  __device__ __forceinline__ unsigned long long weight(float l) const { return token_weight(l, m, scale); }
  __device__ void sync() {
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  }
  __device__ void arrived() {
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  }
  template <typename T>
  __device__ __forceinline__ T* at_first(T* mine) {   // the first CTA's
    return ctas > 1 ? cluster.map_shared_rank(mine, 0) : mine;
  }
  // The run below `top` that a logit falls in: monotone, and the last one is for all that lies further below.
  __device__ static int bin_below(float top, float l) { return l == top ? 0 : (int)fminf((top - l) * 64.0f, (float)(kBins - 1)); }

  // Puts a token on a list if `wanted`; a warp's threads come together.  The list may be too short: its length says so.
  __device__ __forceinline__ void put_into(bool wanted, float l, int id, int* listed, unsigned long long* list, int room = kListed) {
    const unsigned who = __ballot_sync(0xffffffffu, wanted);
    if (who == 0u) return;
    int at = 0;
    if (lane == 0) at = atomicAdd(listed, __popc(who));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
    if (wanted && at < room) list[at] = ((unsigned long long)logit_key(l) << 32) | (unsigned)~id;
  }
  // ... on the first CTA's.
  __device__ __forceinline__ void put(bool wanted, float l, int id) { put_into(wanted, l, id, at_first(&sh.listed), at_first(sh.list)); }
  // Those of four tokens that are not below a bound.
  __device__ __forceinline__ void put_quad(float4 v, float bound, int q, int* listed, unsigned long long* list, int room = kListed) {
    if (!__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound)) return;
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      put_into(v.x >= bound, v.x, first_id + head + 4 * q + e, listed, list, room);
      v.x = v.y, v.y = v.z, v.z = v.w;
    }
  }
  // A token of this thread's among those that do not stand in whole quads, -1 if it has none.
  __device__ __forceinline__ int edge_token() const {
    const int t = threadIdx.x, tail = count - head - 4 * quads;
    return t < head ? t : t - head < tail ? count - tail + t - head : -1;
  }
  __device__ __forceinline__ float4 quad(int q) const { return reinterpret_cast<const float4*>(tokens + head)[q]; }

  // This thread's largest token (NaN is none).  With `asked` (and one CTA) tokens go on the list as they come, those that are not below a bound that so many tokens before are not
  // below; the bound is taken anew when four times (two, where many are asked for) as many tokens have been seen.
  __device__ __forceinline__ void load(int asked) {
    const float nan = __int_as_float(0x7fffffff);
    thread_max = nan;
    constexpr int kFlight = 8;
    float bound = INFINITY;
    int next_bound = kFlight * kFilterThreads;
    for (int q0 = threadIdx.x; q0 - (int)threadIdx.x < quads; q0 += kFlight * kFilterThreads) {
      float4 v[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) v[u] = q0 + u * kFilterThreads < quads ? quad(q0 + u * kFilterThreads) : make_float4(nan, nan, nan, nan);
#pragma unroll
      for (int u = 0; u < kFlight; ++u) thread_max = fmaxf(fmaxf(thread_max, fmaxf(v[u].x, v[u].y)), fmaxf(v[u].z, v[u].w));
      if (asked == 0) continue;
      const int seen = q0 - (int)threadIdx.x + kFlight * kFilterThreads;
      if (seen >= next_bound) {   // (the same for all threads)
        const float largest = block_max(thread_max);
        if (largest > -INFINITY) {   // (while no token is, there is nothing to list and the next batch asks again: a bound has to stand before the first of them is tested)
          bound = key_logit(least_of_maxima(largest, asked, asked).x);
          next_bound = (asked <= 200 ? 4 : 2) * seen;   // (what comes in between has to find room; 256 rows of 128,256, top-k 50: 39.8 us, 41.6 by twos; 160 rows, top-k 300: 103, 71 by twos)
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) put_quad(v[u], bound, q0 + u * kFilterThreads, &sh.listed, sh.early, kEarly);
    }
    const int i = edge_token();
    const float l = i >= 0 ? tokens[i] : nan;
    thread_max = fmaxf(thread_max, l);
    if (asked != 0) put_into(l >= bound, l, first_id + i, &sh.listed, sh.early, kEarly);
  }
  // NaN if all are.
  __device__ __forceinline__ float block_max(float v) {
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, offset));
    if (lane == 0) sh.scan[warp] = __float_as_uint(v);
    __syncthreads();
    v = __uint_as_float((unsigned)sh.scan[lane % kFilterWarps]);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, offset));
    return v;
  }
  // Logits, as keys, that at least `asked` and at least `share` threads' maxima are not below: the least of those that lie in the runs which together hold so many.
  __device__ __forceinline__ uint2 least_of_maxima(float largest, int asked, int share) {
    for (int i = threadIdx.x; i < kBins; i += kFilterThreads) sh.low[i] = 0u;
    if (threadIdx.x < 2) sh.last_run[threadIdx.x] = kBins - 1, sh.least[threadIdx.x] = 0xffffffffu;
    __syncthreads();
    const int bin = bin_below(largest, thread_max);   // (of a thread without a token the last)
    atomicAdd(&sh.low[bin], 1u);
    __syncthreads();
    unsigned of_run[kBinsEach], here = 0u;
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) here += of_run[i] = sh.low[threadIdx.x * kBinsEach + i];
    unsigned upto = here;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += other;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    unsigned before = upto - here;
    for (int w = 0; w < warp; ++w) before += (unsigned)sh.scan[w];
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) {
      if (before < (unsigned)asked && before + of_run[i] >= (unsigned)asked) sh.last_run[0] = threadIdx.x * kBinsEach + i;
      if (before < (unsigned)share && before + of_run[i] >= (unsigned)share) sh.last_run[1] = threadIdx.x * kBinsEach + i;
      before += of_run[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned least = __reduce_min_sync(0xffffffffu, bin <= sh.last_run[i] && sh.last_run[i] < kBins - 1 ? logit_key(thread_max) : 0xffffffffu);
      if (lane == 0) atomicMin(&sh.least[i], least);
    }
    __syncthreads();
    const unsigned none = logit_key(-INFINITY);   // (so few, or so far below, that runs tell no more)
    return make_uint2(sh.least[0] == 0xffffffffu ? none : sh.least[0], sh.least[1] == 0xffffffffu ? none : sh.least[1]);
  }

  // Two numbers of every CTA, in every CTA (a CTA's threads bring the same).  Two places in turn: a CTA is past its reading of one when it brings the one after the next.
  __device__ __forceinline__ const unsigned long long* gather(unsigned long long mine, unsigned long long second) {
    auto& place = sh.gather[gathers ^= 1];
    if (threadIdx.x < ctas) {
      auto* to = ctas > 1 ? cluster.map_shared_rank(&place[0][rank], threadIdx.x) : &place[0][0];
      to[0] = mine;
      to[8] = second;
    }
    sync();
    return place[0];
  }
  // The first token of the order.
  __device__ __forceinline__ int first_of_order() {
    constexpr int kNone = 0x7fffffff, kFlight = 4;
    int id = kNone;
    if (thread_max == m) {   // (who has read such a token looks where it stands)
      for (int q0 = threadIdx.x; q0 < quads && id == kNone; q0 += kFlight * kFilterThreads) {
        float4 v[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; ++f) v[f] = quad(min(q0 + f * kFilterThreads, quads - 1));
#pragma unroll
        for (int f = kFlight - 1; f >= 0; --f) {
          const int at = first_id + head + 4 * min(q0 + f * kFilterThreads, quads - 1);
          id = v[f].x == m ? at : v[f].y == m ? at + 1 : v[f].z == m ? at + 2 : v[f].w == m ? at + 3 : id;
        }
      }
      const int i = edge_token();
      if (i >= 0 && tokens[i] == m) id = min(id, first_id + i);
    }
    id = __reduce_min_sync(0xffffffffu, id);
    if (threadIdx.x == 0) sh.found_id = 0x7fffffff;
    __syncthreads();
    if (lane == 0) atomicMin(&sh.found_id, id);
    __syncthreads();
    const unsigned long long* all = gather(sh.found_id, 0ull);
    for (int c = 0; c < ctas; ++c) id = c == 0 ? (int)all[0] : min(id, (int)all[c]);
    return id;
  }

  // About what a token weighs, of the largest one's weight, and its share of the sum of weights times their distances y = log2 of the weight from the largest.  An eighth of the exact weight's
  // instructions: l - m, the scale and the product are off by 2^-24 each, so a weight by 1.25e-7 |y|, the exponential by 2^-22, a sum of 16 in pairs by 4 * 2^-24, what is left of exact weights below
  // 2^-44 and of |y| above 64 by 2^-25 each, exact weights themselves by 1.5e-7: 1.5e-7 |y| and 8e-7 hold all that.  (NaN counts for 2^-64.)
  __device__ __forceinline__ float about(float l, float slope, float& spread) const {
    const float y = fmaxf((l - m) * slope, -64.0f), w = exp2_approx(y);
    spread = fmaf(w, -y, spread);
    return w;
  }
  __device__ __forceinline__ float about(float4 v, float slope, float& spread) const {
    return (about(v.x, slope, spread) + about(v.y, slope, spread)) + (about(v.z, slope, spread) + about(v.w, slope, spread));
  }
  __device__ static unsigned long long in_units(float w) { return (unsigned long long)(w * (float)(1ull << kWeightBits)); }
  __device__ static unsigned long long spread_in_units(float spread) { return (unsigned long long)(spread * 1048576.0f); }
  // How far what tokens weigh about, in units of 2^-44, is off what they weigh at most.
  __device__ static unsigned long long off_at_most(unsigned long long about, unsigned long long spread) {
    return (unsigned long long)((double)about * 8e-7 + ((double)spread / 1048576.0 + 0.01) * (1.5e-7 * (double)(1ull << kWeightBits))) + 1ull;
  }
  // Lists the tokens that are not below the bound; with `weights` about what all tokens weigh, this thread's share of it.  Whether top_p's border lies on the same token for all totals in between
  // is seen when the list is in order; if not, exact weights tell.
  __device__ __forceinline__ void list_from(float bound, bool weights, unsigned long long& mine, float& spread) {
    const float nan = __int_as_float(0x7fffffff), slope = (float)scale.c;
    constexpr int kFlight = 4;
    for (int q0 = threadIdx.x; q0 - (int)threadIdx.x < quads; q0 += kFlight * kFilterThreads) {
      float4 v[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) v[u] = q0 + u * kFilterThreads < quads ? quad(q0 + u * kFilterThreads) : make_float4(nan, nan, nan, nan);
      if (weights) {
        static_assert(kFlight == 4, "sums of 16");
        mine += in_units((about(v[0], slope, spread) + about(v[1], slope, spread)) + (about(v[2], slope, spread) + about(v[3], slope, spread)));
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) put_quad(v[u], bound, q0 + u * kFilterThreads, at_first(&sh.listed), at_first(sh.list));
    }
    const int i = edge_token();
    const float l = i >= 0 ? tokens[i] : nan;
    if (weights) mine += in_units(about(l, slope, spread));
    put(l >= bound, l, first_id + i);
  }

  // The row's token if its first top_k tokens (or all that min_p leaves, or, where the weight of all tokens lies between `least` and `most`, all that top_p leaves) are on the list; by the
  // first CTA.  Where the list's weight does not reach top_p of all tokens' kListTooShort, where it depends on what they weigh exactly kUnsure.
  __device__ __forceinline__ int choose_from_list(int top_k, float top_p, unsigned long long least, unsigned long long most, float u) {
    const int number = min(top_k, sh.listed), mine = threadIdx.x;
    const unsigned long long token = sort_falling(sh.list[mine], sh.listed, sh.exchange);
    const unsigned long long w = mine < number ? weight(key_logit((unsigned)(token >> 32))) : 0ull;
    unsigned long long all, of_kept;
    const unsigned long long before = block_prefix(w, sh.scan, all);
    if (most == 0ull) least = most = all;
    else if (all < wanted_of(top_p, least)) return kListTooShort;
    else if (all < wanted_of(top_p, most)) return kUnsure;
    // kept: in front of which top_p has not been reached, heavy enough; the first always
    const bool heavy = mine < number && w >= floor_weight;
    const int many = __syncthreads_count(mine == 0 || (heavy && before < wanted_of(top_p, least)));
    if (least != most && __syncthreads_count(mine == 0 || (heavy && before < wanted_of(top_p, most))) != many) return kUnsure;
    // in order of ids (the lower one's complement is the larger), the weight behind the id
    const unsigned long long by_id = sort_falling(((unsigned long long)((unsigned)token & (kFilterMaxVocab - 1)) << (kWeightBits + 1)) | w, many, sh.exchange);
    const unsigned long long kept_weight = mine < many ? by_id & ((2ull << kWeightBits) - 1ull) : 0ull;
    const unsigned long long start = block_prefix(kept_weight, sh.scan, of_kept), target = target_of(u, of_kept);
    if (target >= start && target < start + kept_weight) sh.found_id = (int)(~(unsigned)(by_id >> (kWeightBits + 1)) & (kFilterMaxVocab - 1));
    __syncthreads();
    return sh.found_id;
  }
  // What top_p of a total comes to.
  __device__ static unsigned long long wanted_of(float top_p, unsigned long long total) {
    return top_p < 1.0f ? max(1ull, min(total, (unsigned long long)ceil((double)top_p * (double)total))) : ~0ull;
  }
  __device__ static unsigned long long target_of(float u, unsigned long long total) {
    const unsigned long long target = u > 0.0f ? (unsigned long long)((double)fminf(u, 1.0f) * (double)total) : 0ull;
    return target >= total ? total - 1ull : target;
  }

  // --- where the list does not do ---------------------------------------------------------------
  // f(logit, id) for all tokens, a warp's threads together; where there is no token NaN and an id that is none.
  template <typename F>
  __device__ __forceinline__ void for_tokens(F f) {
    const float nan = __int_as_float(0x7fffffff);
    constexpr int kFlight = 4;
    for (int q0 = threadIdx.x; q0 - (int)threadIdx.x < quads; q0 += kFlight * kFilterThreads) {
      float4 v[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) v[u] = q0 + u * kFilterThreads < quads ? quad(q0 + u * kFilterThreads) : make_float4(nan, nan, nan, nan);
#pragma unroll 1
      for (int u = 0; u < kFlight; ++u) {
        const int q = q0 + u * kFilterThreads, id = q < quads ? first_id + head + 4 * q : -8;
        f(v[0].x, id);
        f(v[0].y, id + 1);
        f(v[0].z, id + 2);
        f(v[0].w, id + 3);
#pragma unroll
        for (int other = 0; other + 1 < kFlight; ++other) v[other] = v[other + 1];
      }
    }
    const int i = edge_token();
    f(i >= 0 ? tokens[i] : nan, i >= 0 ? first_id + i : -1);
  }
  __device__ __forceinline__ void add_to_bin(int bin, unsigned long long v) {
    if (v == 0ull) return;
    const unsigned part = (unsigned)v, before = atomicAdd(&sh.low[bin], part);
    const unsigned rest = (unsigned)(v >> 32) + (before + part < before ? 1u : 0u);
    if (rest != 0u) atomicAdd(&sh.high[bin], rest);
  }
  // The shortest prefix of the order that brings `wanted` tokens, or `share` of the weight of all that `within` holds.
  __device__ __forceinline__ Border find(const Border& within, unsigned long long wanted, bool weights, float share) {
    unsigned from = 0u, to = 0xffffffffu;   // keys among which the border lies (from level 1 on)
    int shift = 0;
#pragma unroll 1
    for (int level = 0;; ++level) {
      // the run of a token at this level, -1 if it does not count
      auto run_of = [&](float l, int id) {
        const unsigned key = logit_key(l);
        if (id < 0 || !within.holds(key, id)) return -1;
        if (level == 0) return bin_below(m, l);
        return key >= from && key <= to ? (int)((to - key) >> shift) : -1;
      };
      for (int i = threadIdx.x; i < kBins; i += kFilterThreads) sh.low[i] = sh.high[i] = 0u;
      __syncthreads();
      for_tokens([&](float l, int id) {
        const int run = run_of(l, id);
        if (run >= 0) add_to_bin(run, weights ? weight(l) : 1ull);
      });
      sync();
      if (rank == 0) {   // what lies in the cluster's bins, those of this thread and those before
        unsigned long long of_bin[kBinsEach], sum = 0ull, all;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) {
          of_bin[i] = 0ull;
          for (int c = 0; c < ctas; ++c) {
            const unsigned* low = (ctas > 1 ? cluster.map_shared_rank(sh.low, c) : sh.low) + threadIdx.x * kBinsEach + i;
            of_bin[i] += ((unsigned long long)low[kBins] << 32) + low[0];   // (the upper words lie behind the lower ones)
          }
          sum += of_bin[i];
        }
        unsigned long long before = block_prefix(sum, sh.scan, all);
        if (level == 0 && weights) wanted = max(1ull, min(all, (unsigned long long)ceil((double)share * (double)all)));
        before += level == 0 ? 0ull : sh.above;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) {
          if (before < wanted && before + of_bin[i] >= wanted) {
            sh.bin = threadIdx.x * kBinsEach + i;
            sh.above = before;
            sh.wanted = wanted;
          }
          before += of_bin[i];
        }
        if (threadIdx.x == 0) sh.listed = 0;
      }
      sync();
      const int border_run = *at_first(&sh.bin);
      wanted = *at_first(&sh.wanted);
      unsigned lowest = 0xffffffffu, highest = 0u;
      for_tokens([&](float l, int id) {
        const bool in_run = run_of(l, id) == border_run;
        if (in_run) lowest = min(lowest, logit_key(l)), highest = max(highest, logit_key(l));
        put(in_run, l, id);
      });
      lowest = __reduce_min_sync(0xffffffffu, lowest);
      highest = __reduce_max_sync(0xffffffffu, highest);
      if (lane == 0) sh.scan[warp] = ((unsigned long long)highest << 32) | lowest;
      __syncthreads();
      for (int w = 0; w < kFilterWarps; ++w) lowest = min(lowest, (unsigned)sh.scan[w]), highest = max(highest, (unsigned)(sh.scan[w] >> 32));
      const unsigned long long* all = gather(lowest, highest);
      if (*at_first(&sh.listed) <= kListed) {
        if (rank == 0) border_of_list(wanted, weights);
        sync();
        return Border{*at_first(&sh.found_key), *at_first(&sh.found_id)};
      }
      from = 0xffffffffu, to = 0u;
      for (int c = 0; c < ctas; ++c) from = min(from, (unsigned)all[c]), to = max(to, (unsigned)all[8 + c]);
      if (from == to) return border_of_equals(within, to, wanted, weights);
      shift = max(0, 32 - __clz(to - from) - kBinBits);
      sync();   // (all have read the list's length before the next level clears it)
    }
  }
  // Where on the first CTA's list (the border's run) the border lies.
  __device__ __forceinline__ void border_of_list(unsigned long long wanted, bool weights) {
    const int listed = sh.listed;
    const unsigned long long token = sort_falling(sh.list[threadIdx.x], listed, sh.exchange);
    const unsigned long long w = (int)threadIdx.x >= listed ? 0ull : weights ? weight(key_logit((unsigned)(token >> 32))) : 1ull;
    unsigned long long all;
    const unsigned long long before = sh.above + block_prefix(w, sh.scan, all);
    if (before < wanted && before + w >= wanted) {
      sh.found_key = (unsigned)(token >> 32);
      sh.found_id = (int)~(unsigned)token;
    }
  }
  // The border among more tokens of one key than the list holds: so many of them, in order of ids, as are still wanted.
  __device__ __forceinline__ Border border_of_equals(const Border& within, unsigned key, unsigned long long wanted, bool weights) {
    const unsigned long long each = weights ? weight(key_logit(key)) : 1ull, above = *at_first(&sh.above);
    const unsigned long long number = (wanted - above + each - 1ull) / each;   // (a border in weight lies where there is some)
    const int segment = (count + kFilterWarps - 1) / kFilterWarps, begin = min(count, warp * segment), end = min(count, begin + segment);
    unsigned mine = 0u;
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      mine += __popc(__ballot_sync(0xffffffffu, i < end && logit_key(tokens[i]) == key && within.holds(key, first_id + i)));
    }
    unsigned long long all, before = block_prefix(lane == 0 ? (unsigned long long)mine : 0ull, sh.scan, all);
    before = __shfl_sync(0xffffffffu, before, 0);
    const unsigned long long* of_cta = gather(all, 0ull);
    for (int c = 0; c < rank; ++c) before += of_cta[c];
    if (before < number && before + mine >= number) {
      unsigned left = (unsigned)(number - before);
      for (int i0 = begin; i0 < end; i0 += 32) {
        const int i = i0 + lane;
        const unsigned who = __ballot_sync(0xffffffffu, i < end && logit_key(tokens[i]) == key && within.holds(key, first_id + i));
        const unsigned here = __popc(who);
        if (left <= here) {
          if ((who >> lane & 1u) && __popc(who & ((1u << lane) - 1u)) == (int)left - 1) *at_first(&sh.found_id) = first_id + i;
          break;
        }
        left -= here;
      }
    }
    sync();
    return Border{key, *at_first(&sh.found_id)};
  }
  // The token that the number falls on among all of them, in order of ids: from exact weights, or from what they weigh about, and -1 then if it lies too near another token for that.
  template <bool EXACT>
  __device__ __forceinline__ int draw_from_all(float u) {
    const float slope = (float)scale.c, nan = __int_as_float(0x7fffffff);
    float spread = 0.0f;
    auto of_token = [&](float l) { return EXACT ? weight(l) : in_units(about(l, slope, spread)); };
    const int segment = (quads + kFilterWarps - 1) / kFilterWarps, begin = min(quads, warp * segment), end = min(quads, begin + segment);   // as below
    unsigned long long mine = 0ull;
    constexpr int kFlight = 4;
    for (int q0 = begin + lane; q0 < end; q0 += 32 * kFlight) {
      float4 v[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) v[f] = q0 + 32 * f < end ? quad(q0 + 32 * f) : make_float4(nan, nan, nan, nan);
      static_assert(kFlight == 4, "sums of 16");
      if constexpr (EXACT) {
#pragma unroll 1
        for (int f = 0; f < kFlight; ++f) {
          mine += (weight(v[0].x) + weight(v[0].y)) + (weight(v[0].z) + weight(v[0].w));
#pragma unroll
          for (int other = 0; other + 1 < kFlight; ++other) v[other] = v[other + 1];
        }
      } else {
        mine += in_units((about(v[0], slope, spread) + about(v[1], slope, spread)) + (about(v[2], slope, spread) + about(v[3], slope, spread)));
      }
    }
    const int first = warp == 0 ? 0 : head + 4 * begin, last = warp == kFilterWarps - 1 ? count : head + 4 * end;   // this warp's tokens
    if (warp == 0 && lane < head) mine += of_token(tokens[lane]);
    if (warp == kFilterWarps - 1 && head + 4 * quads + lane < count) mine += of_token(tokens[head + 4 * quads + lane]);
    mine = warp_sum_u64(mine);
    unsigned long long far = warp_sum_u64(spread_in_units(spread));
    if (lane == 0) sh.exchange[0][warp] = far;
    if (threadIdx.x == 0) sh.found_id = -1;
    unsigned long long all, before = block_prefix(lane == 0 ? mine : 0ull, sh.scan, all);
    before = __shfl_sync(0xffffffffu, before, 0);
    far = 0ull;
    for (int w = 0; w < kFilterWarps; ++w) far += sh.exchange[0][w];
    const unsigned long long* of_cta = gather(all, far);
    unsigned long long total = 0ull, start = 0ull;
    far = 0ull;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank) start += of_cta[c];
      total += of_cta[c], far += of_cta[8 + c];
    }
    // The number's place is off by so much at most, and so is where a token begins or ends (every token in front of it counts once).
    const unsigned long long target = target_of(u, total), off = EXACT ? 0ull : 2ull * off_at_most(total, far) + 8ull;
    if (target >= start && target < start + all) {
      if (lane == 0 && target >= start + before && target < start + before + mine) sh.last_run[0] = first, sh.last_run[1] = last, sh.above = start + before;
      __syncthreads();
      const int from = sh.last_run[0], to = sh.last_run[1], each = (to - from + kFilterThreads - 1) / kFilterThreads;
      const int a = min(to, from + (int)threadIdx.x * each), b = min(to, a + each);
      unsigned long long part = 0ull, sum;
      for (int i = a; i < b; ++i) part += of_token(tokens[i]);
      unsigned long long running = sh.above + block_prefix(part, sh.scan, sum);
      if (target >= running && target < running + part) {
        for (int i = a; i < b; ++i) {
          const unsigned long long w = of_token(tokens[i]);
          if (target >= running + off && target + off < running + w) *at_first(&sh.found_id) = first_id + i;   // (a token at most)
          running += w;
        }
      }
    }
    sync();
    return *at_first(&sh.found_id);
  }
  // The token that the number falls on among the kept ones, in order of ids.
  __device__ __forceinline__ int draw(const Border& kept, float u) {
    auto kept_weight = [&](float l, int i) {
      const unsigned long long w = weight(l);
      return kept.holds(logit_key(l), first_id + i) && w >= floor_weight ? w : 0ull;
    };
    // consecutive quads per warp; what stands in front of the first and behind the last one is the first and the last warp's
    const int segment = (quads + kFilterWarps - 1) / kFilterWarps, begin = min(quads, warp * segment), end = min(quads, begin + segment);
    const float nan = __int_as_float(0x7fffffff);
    unsigned long long mine = 0ull;
    constexpr int kFlight = 4;
    for (int q0 = begin + lane; q0 < end; q0 += 32 * kFlight) {
      float4 v[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) v[f] = q0 + 32 * f < end ? quad(q0 + 32 * f) : make_float4(nan, nan, nan, nan);
#pragma unroll 1
      for (int f = 0; f < kFlight; ++f) {
        const int i = head + 4 * (q0 + 32 * f);
        mine += (kept_weight(v[0].x, i) + kept_weight(v[0].y, i + 1)) + (kept_weight(v[0].z, i + 2) + kept_weight(v[0].w, i + 3));
#pragma unroll
        for (int other = 0; other + 1 < kFlight; ++other) v[other] = v[other + 1];
      }
    }
    const int first = warp == 0 ? 0 : head + 4 * begin, last = warp == kFilterWarps - 1 ? count : head + 4 * end;   // this warp's tokens
    if (warp == 0 && lane < head) mine += kept_weight(tokens[lane], lane);
    if (warp == kFilterWarps - 1 && head + 4 * quads + lane < count) mine += kept_weight(tokens[head + 4 * quads + lane], head + 4 * quads + lane);
    mine = warp_sum_u64(mine);
    unsigned long long all, before = block_prefix(lane == 0 ? mine : 0ull, sh.scan, all);
    before = __shfl_sync(0xffffffffu, before, 0);
    const unsigned long long* of_cta = gather(all, 0ull);
    unsigned long long total = 0ull, start = 0ull;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank) start += of_cta[c];
      total += of_cta[c];
    }
    const unsigned long long target = target_of(u, total);
    if (target >= start && target < start + all) {   // in this CTA: all its threads look through the warp's tokens that it falls on
      if (lane == 0 && target >= start + before && target < start + before + mine) sh.last_run[0] = first, sh.last_run[1] = last, sh.above = start + before;
      __syncthreads();
      const int from = sh.last_run[0], to = sh.last_run[1], each = (to - from + kFilterThreads - 1) / kFilterThreads;
      const int a = min(to, from + (int)threadIdx.x * each), b = min(to, a + each);
      unsigned long long part = 0ull, sum;
      for (int i = a; i < b; ++i) part += kept_weight(tokens[i], i);
      unsigned long long running = sh.above + block_prefix(part, sh.scan, sum);
      if (target >= running && target < running + part) {
        int i = a;
        for (; i < b; ++i) {
          running += kept_weight(tokens[i], i);
          if (target < running) break;
        }
        *at_first(&sh.found_id) = first_id + i;
      }
    }
    sync();
    return sh.found_id;
  }
};

__global__ void __launch_bounds__(kFilterThreads, 2)
    sample_filtered_kernel(const float* __restrict__ logits, long long row_stride, int all_rows, int vocab, int slice, const int* __restrict__ rows, const float* __restrict__ temperature,
                           const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniforms,
                           int* __restrict__ out) {
  __shared__ FilterShared shared;
  const int ctas = cooperative_groups::this_cluster().num_blocks(), set = blockIdx.x / ctas;
  grid_dependency_wait();
  const int index = rows != nullptr ? rows[set] : set;
  if (index < 0 || index >= all_rows) return;   // (the whole cluster)
  const float t = temperature[set], p = top_p[set], smallest = min_p[set], u = uniforms[set];
  const int k = top_k[set];
  if (threadIdx.x == 0) shared.listed = 0;
  __syncthreads();
  RowFilter filter(shared, logits + (size_t)index * row_stride, vocab, slice);
  filter.arrive();
  const int token = filter.choose(t, k, p, smallest, u);
  if (cooperative_groups::this_cluster().block_rank() == 0) {
    if (threadIdx.x == 0) out[index] = token;
    if (ctas > 1) cooperative_groups::this_cluster().sync();   // the others leave when they are done; this CTA's memory stays until they have (who has left is not waited for)
  }
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
  // CTAs of a row's cluster, with at least 8,192 tokens each where there are two and more: one per SM in all, or two if each has 16,384 tokens (clusters of four and eight do not fill every
  // SM: nine tenths of that).  us, by halving the CTAs: 120 rows of 32,000 without options 12.9 -> 9.5 (one per SM), 40 rows of 128,256 under top-p 26.8 -> 29.4 (one per SM; two are taken); 74 rows of 128,256
  // under top-p in 296 CTAs 43.5, in 148 30.2.  The rule knows sizes only (the options lie on the device) and was fitted to rows under top-p.  Its steps show with every option where rows lose a CTA:
  // 148 -> 149 rows of 128,256 take 47 -> 61 us without options, 51 -> 64 under top-p, 35.2 -> 35.5 with top-k 50.
  const int sms = device_sm_count();
  int ctas = 1;
  while (ctas < 8 && vocab > ctas * 8192) {
    const int next = 2 * ctas, room = vocab < next * 16384 ? sms : next >= 4 ? sms * 9 / 5 : sms * 2;
    if ((long long)count * next > room) break;
    ctas = next;
  }
  const int slice = ((vocab + ctas - 1) / ctas + 3) & ~3;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)count * ctas);
  config.blockDim = dim3(kFilterThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = ctas;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  static const bool pdl = [] {
    const char* v = std::getenv("TLIE_PDL");
    return !(v && v[0] == '0');
  }();
  config.numAttrs = pdl ? 2 : 1;
  return (int)cudaLaunchKernelEx(&config, sample_filtered_kernel, logits, row_stride, all_rows, vocab, slice, rows, temperature, top_k, top_p, min_p, uniforms, out);
}

TLIE_EXPORT int tlie_uniforms(const long long* seeds, const long long* counters, float* out, int count, cudaStream_t stream) {
  if (count <= 0) return 0;
  uniforms_kernel<<<(count + 255) / 256, 256, 0, stream>>>(seeds, counters, out, count);
  return (int)cudaGetLastError();
}
