// Paged grouped-query attention for a batch whose requests share their first `shared` cached keys (answers to one prompt, questions behind one
// system prompt): the general kernel, for 32-bit and bfloat16 rows, any head size up to 256 and any page size.
//
// Row t of the step, of entry b at position p, and query head h (key/value head g = h / group) see keys j <= p:
//   out = sum_j e^(scale q.k_j - m) v_j / sum_j e^(scale q.k_j - m)
// Keys j < shared lie in the pages that row 0 of the block table names (every entry's row names the same), keys from there on in those of row b.
// The sum is taken in parts, (m, l, o) = (largest score, sum of weights, weighted sum of values) each, and the parts are brought together:
// with M = max m_i, out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i (scores in units of log2).  Parts of the prefix are worked out
// for all rows of the step at once, so that its keys and values are read once per 32 rows and not once per request; parts of an entry's own keys for its rows.
//
// A CTA owns one key/value head, 32 (row, head) pairs and a run of keys, which it copies to shared memory 32 at a time, the next ones while it works on these.
// Scores (32 x 32) and weighted values (32 x head size) are register tiles of two pairs per thread: 32 multiply-adds for six 16-byte reads of shared memory, 64 for
// ten.  (With one thread to a score and one to a channel the four rows below took 104 us.)  All sums are
// 32-bit.  Bound by reads of shared memory where there are many rows (480 rows, 32 heads of 64 over 4, 900 shared and up to 200 own keys: 218 us for 3.7 GFLOP, shared memory busy 60% of the
// time), by the chain of a chunk's steps where there are few (so runs are short there): 4 rows of the same heads behind 500 keys take 12 us, 5 of them for joining the parts.
// bfloat16 heads of other sizes than 64 and 128 come here too and are worked out on 32-bit numbers: 8 rows, 32 heads of 96 over 8, 1,024 shared and 30 own keys: 23 us; 64 rows, 700 and 200: 225, where the
// kernel for single rows that shares nothing (attention_decode.cu, head sizes up to 128) takes 34; 16 rows, 16 heads of 256, 1,000 and 100: 383, where the general kernel that shares nothing takes 1,120.
#include "common.cuh"
#include "mma_utils.cuh"
#include "shared_memory_limit.cuh"

namespace tlie {

constexpr int kPairs = 32;         // (row, head) pairs of a CTA
constexpr int kPairThreads = 128;  // 16 times two pairs, 8 times four keys, or the value's channels in eight parts
constexpr int kChunk = 32;         // keys in shared memory at a time
constexpr float kToLog2 = 1.4426950408889634f;
constexpr int kBadPage = 8;        // the bit of the device's error word

struct SharedPrefixParams {
  const void* q;
  long long q_row_stride;
  const void* pages;
  int num_pages;
  const int* positions;
  const int* seq_starts;
  const int* block_table;
  int table_stride;
  void* out;
  float* part_o;        // [rows, q heads, parts, head size]
  float2* part_ml;      // [rows, q heads, parts]: largest score in units of log2, sum of weights
  int rows, entries, q_heads, kv_heads, head_dim, page_size, shared;
  float scale;
  int prefix_parts, own_parts;
  int* error_flag;
};

// The page of logical page `index` of a table row: what lies outside the table or the pool is reported, and page 0 read in its place.
__device__ __forceinline__ int page_of(const SharedPrefixParams& p, const int* table, int index) {
  const int page = index < p.table_stride ? table[index] : -1;
  if ((unsigned)page < (unsigned)p.num_pages) return page;
  atomicOr(p.error_flag, kBadPage);
  return 0;
}

__device__ __forceinline__ void dot4(float& acc, float4 a, float4 b) { acc = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, acc)))); }
__device__ __forceinline__ void add4(float4& acc, float w, float4 v) {
  acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
}

// MAX_DIM: 64, 128 or 256, the head size rounded up.
template <typename T, int MAX_DIM>
__global__ void __launch_bounds__(kPairThreads) shared_prefix_generic_kernel(SharedPrefixParams p, int tiles_of_all) {
  extern __shared__ __align__(16) float smem[];
  constexpr int kQuads = MAX_DIM / 32;         // four channels each, of this thread's share of a value
  const int D = p.head_dim, key_row = D + 4;   // four floats more: threads that read 16 bytes of eight keys' rows, or of every other of eight queries', touch different banks
  float* q_smem = smem;                        // [pairs][D + 4]
  float* w_smem = q_smem + kPairs * key_row;   // [pairs][keys + 4]
  constexpr int kWeightRow = kChunk + 4;
  float* chunks = w_smem + kPairs * kWeightRow;   // twice [keys][D + 4] of keys and [keys][D] of values
  const int chunk_floats = kChunk * key_row + kChunk * D;
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 3, tx = threadIdx.x & 7;
  const int kvh = blockIdx.y, group = p.q_heads / p.kv_heads;
  grid_dependency_wait();
  const int first_row = max(0, p.seq_starts[0]), end_row = min(p.seq_starts[p.entries], p.rows);
  // the prefix's parts, `tiles_of_all` CTAs each, then those of the entries' own keys with a CTA more per entry
  const bool of_prefix = blockIdx.x < (unsigned)tiles_of_all * p.prefix_parts;
  const unsigned number = of_prefix ? blockIdx.x : blockIdx.x - (unsigned)tiles_of_all * p.prefix_parts, tiles_here = of_prefix ? tiles_of_all : tiles_of_all + p.entries;
  const int which = (int)(number / tiles_here), tile = (int)(number % tiles_here), part = of_prefix ? which : p.prefix_parts + which;

  // which pairs: consecutive ones of all rows, or of one entry's rows
  int row0 = 0, pairs = 0, entry = 0;
  long long pair0 = (long long)tile * kPairs;
  if (of_prefix) {
    const long long all = (long long)(end_row - first_row) * group;
    if (pair0 >= all) return;
    row0 = first_row;
    pairs = (int)min((long long)kPairs, all - pair0);
  } else {   // the entry that this tile number falls to, counting every entry's tiles: 32 entries at a time
    int tiles_before = 0;
    for (int e0 = 0; e0 < p.entries; e0 += 32) {
      const int e = e0 + lane;
      int begin = 0, end = 0;
      if (e < p.entries) {
        begin = max(0, p.seq_starts[e]);
        end = min(p.rows, p.seq_starts[e + 1]);
      }
      const int tiles = end > begin ? (int)(((long long)(end - begin) * group + kPairs - 1) / kPairs) : 0;
      int upto = tiles;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if (lane >= offset) upto += other;
      }
      const unsigned past = __ballot_sync(0xffffffffu, tiles_before + upto > tile);
      if (past != 0u) {
        const int at = __ffs(past) - 1;
        entry = e0 + at;
        const int before = tiles_before + __shfl_sync(0xffffffffu, upto - tiles, at);
        row0 = __shfl_sync(0xffffffffu, begin, at);
        const int rows_here = __shfl_sync(0xffffffffu, end, at) - row0;
        pair0 = (long long)(tile - before) * kPairs;
        pairs = (int)min((long long)kPairs, (long long)rows_here * group - pair0);
        break;
      }
      tiles_before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (pairs <= 0) return;
  }
  // pair i of the tile: row and head, in lane i; `at` is the pair's place among all pairs of a row and a query head
  const int before_first = (int)(pair0 % group) + lane;
  const int row = row0 + (int)(pair0 / group) + before_first / group, head = kvh * group + before_first % group;
  const long long at_lane = (long long)row * p.q_heads + head;

  const int* table = p.block_table + (size_t)entry * p.table_stride;
  const long long room = (long long)p.table_stride * p.page_size;
  // keys a pair sees in this kind of part: below the result; lane i has pair i's
  int limit = 0;
  if (lane < pairs) {
    long long seen = (long long)p.positions[row] + 1;
    if (seen > room) {
      if (threadIdx.x < 32) atomicOr(p.error_flag, kBadPage);
      seen = room;
    }
    limit = (int)max(0ll, of_prefix ? min(seen, (long long)p.shared) : seen);
  }
  const int last = __reduce_max_sync(0xffffffffu, limit);
  const int limits[2] = {__shfl_sync(0xffffffffu, limit, 2 * ty), __shfl_sync(0xffffffffu, limit, 2 * ty + 1)};
  const int lowest = __reduce_min_sync(0xffffffffu, lane < pairs ? limit : 0x7fffffff);
  const int from = of_prefix ? 0 : p.shared;
  const int all_chunks = last > from ? (last - from + kChunk - 1) / kChunk : 0;
  const int parts_here = of_prefix ? p.prefix_parts : p.own_parts;
  const int chunk_begin = (int)((long long)all_chunks * which / parts_here), chunk_end = (int)((long long)all_chunks * (which + 1) / parts_here);

  const size_t plane = (size_t)p.kv_heads * p.page_size * D;
  // The keys and values of a chunk: 16 bytes a copy.  Places past the last key become zeros.
  auto fetch = [&](int chunk) {
    constexpr int kEach = 16 / (int)sizeof(T);
    float* k_smem = chunks + (chunk & 1) * chunk_floats;
    float* v_smem = k_smem + kChunk * key_row;
    const int j = threadIdx.x >> 2, key = from + chunk * kChunk + j;   // four threads a key
    const bool there = key < last;
    const T* token = (const T*)p.pages;
    if (there) token += (size_t)page_of(p, table, key / p.page_size) * 2 * plane + ((size_t)kvh * p.page_size + key % p.page_size) * D;
#pragma unroll 4
    for (int d = (threadIdx.x & 3) * kEach; d < D; d += 4 * kEach) {
      const T* from_page = there ? token + d : token;
      if constexpr (sizeof(T) == 4) {
        cp_async_16(k_smem + j * key_row + d, from_page, there);
        cp_async_16(v_smem + j * D + d, there ? from_page + plane : from_page, there);
      } else {
        uint4 k = make_uint4(0, 0, 0, 0), v = k;
        if (there) k = *reinterpret_cast<const uint4*>(from_page), v = *reinterpret_cast<const uint4*>(from_page + plane);
        const unsigned k_words[4] = {k.x, k.y, k.z, k.w}, v_words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          k_smem[j * key_row + d + 2 * w] = __uint_as_float(k_words[w] << 16), k_smem[j * key_row + d + 2 * w + 1] = __uint_as_float(k_words[w] & 0xffff0000u);
          v_smem[j * D + d + 2 * w] = __uint_as_float(v_words[w] << 16), v_smem[j * D + d + 2 * w + 1] = __uint_as_float(v_words[w] & 0xffff0000u);
        }
      }
    }
    cp_async_commit();
  };
  if (chunk_begin < chunk_end) fetch(chunk_begin);
  const long long q_lane = (long long)row * p.q_row_stride + (long long)head * D;
#pragma unroll
  for (int i = 0; i < kPairs / 4; ++i) {   // a warp brings eight queries
    const int pair = (threadIdx.x >> 5) * (kPairs / 4) + i;
    const T* q = (const T*)p.q + __shfl_sync(0xffffffffu, q_lane, pair);
#pragma unroll
    for (int d = 0; d < MAX_DIM; d += 32)
      if (d + lane < D) q_smem[pair * key_row + d + lane] = pair < pairs ? to_float(q[d + lane]) * p.scale * kToLog2 : 0.0f;
  }
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};   // of pairs 2 ty and 2 ty + 1, the same in their eight threads
  float4 acc[2][kQuads];                                          // channels 4 (tx + 8 c)
#pragma unroll
  for (int c = 0; c < kQuads; ++c) acc[0][c] = acc[1][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int chunk = chunk_begin; chunk < chunk_end; ++chunk) {
    if (chunk + 1 < chunk_end) {
      fetch(chunk + 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    const float* k_smem = chunks + (chunk & 1) * chunk_floats;
    const float* v_smem = k_smem + kChunk * key_row;
    const int key0 = from + chunk * kChunk;
    float score[2][4];   // pair 2 ty + r, key tx + 8 i
#pragma unroll
    for (int i = 0; i < 4; ++i) score[0][i] = score[1][i] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      const float4 q0 = *reinterpret_cast<const float4*>(q_smem + 2 * ty * key_row + d), q1 = *reinterpret_cast<const float4*>(q_smem + (2 * ty + 1) * key_row + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 k = *reinterpret_cast<const float4*>(k_smem + (tx + 8 * i) * key_row + d);
        dot4(score[0][i], q0, k);
        dot4(score[1][i], q1, k);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float here = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (key0 + tx + 8 * i >= limits[r]) score[r][i] = -INFINITY;
        here = fmaxf(here, score[r][i]);
      }
#pragma unroll
      for (int other = 1; other < 8; other <<= 1) here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, other));
      const float reference = fmaxf(top[r], here), base = reference == -INFINITY ? 0.0f : reference;
      const float shrink = exp2f(top[r] - base);
      top[r] = reference;
      float more = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = exp2f(score[r][i] - base);
        w_smem[(2 * ty + r) * kWeightRow + tx + 8 * i] = w;
        more += w;
      }
#pragma unroll
      for (int other = 1; other < 8; other <<= 1) more += __shfl_xor_sync(0xffffffffu, more, other);
      sum[r] = fmaf(sum[r], shrink, more);
#pragma unroll
      for (int c = 0; c < kQuads; ++c) acc[r][c].x *= shrink, acc[r][c].y *= shrink, acc[r][c].z *= shrink, acc[r][c].w *= shrink;
    }
    __syncwarp();   // (a pair's weights are its own eight threads')
    const float* w0_row = w_smem + 2 * ty * kWeightRow;
    const float* w1_row = w0_row + kWeightRow;
    if (key0 + kChunk <= lowest) {
#pragma unroll 2
      for (int j = 0; j < kChunk; j += 4) {
        const float4 w0 = *reinterpret_cast<const float4*>(w0_row + j), w1 = *reinterpret_cast<const float4*>(w1_row + j);
#pragma unroll
        for (int c = 0; c < kQuads; ++c) {
          const int d = 4 * (tx + 8 * c);
          if (d >= D) break;
          const float4 v0 = *reinterpret_cast<const float4*>(v_smem + j * D + d), v1 = *reinterpret_cast<const float4*>(v_smem + (j + 1) * D + d);
          const float4 v2 = *reinterpret_cast<const float4*>(v_smem + (j + 2) * D + d), v3 = *reinterpret_cast<const float4*>(v_smem + (j + 3) * D + d);
          add4(acc[0][c], w0.x, v0), add4(acc[0][c], w0.y, v1), add4(acc[0][c], w0.z, v2), add4(acc[0][c], w0.w, v3);
          add4(acc[1][c], w1.x, v0), add4(acc[1][c], w1.y, v1), add4(acc[1][c], w1.z, v2), add4(acc[1][c], w1.w, v3);
        }
      }
    } else {
      // Only keys that a pair sees are added: what lies in another's later places (it may be no number) must not reach it through a weight of zero.
#pragma unroll 1
      for (int j = 0; j < kChunk; ++j)
#pragma unroll
        for (int c = 0; c < kQuads; ++c) {
          const int d = 4 * (tx + 8 * c);
          if (d >= D) break;
          const float4 v = *reinterpret_cast<const float4*>(v_smem + j * D + d);
          if (key0 + j < limits[0]) add4(acc[0][c], w0_row[j], v);
          if (key0 + j < limits[1]) add4(acc[1][c], w1_row[j], v);
        }
    }
    __syncthreads();
  }
  const int parts = p.prefix_parts + p.own_parts;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = 2 * ty + r;
    const size_t at = (size_t)__shfl_sync(0xffffffffu, at_lane, i) * parts + part;
    if (i >= pairs) continue;
    if (tx == 0) p.part_ml[at] = make_float2(top[r], sum[r]);
#pragma unroll
    for (int c = 0; c < kQuads; ++c)
      if (4 * (tx + 8 * c) < D) *reinterpret_cast<float4*>(p.part_o + at * D + 4 * (tx + 8 * c)) = acc[r][c];
  }
}

// One CTA per (row, head): the parts brought together.  A thread has four channels of every so many-th part, four parts' loads in flight; a row that sees no
// key gives zeros.
constexpr int kMergeThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kMergeThreads) shared_prefix_merge_kernel(SharedPrefixParams p) {
  __shared__ float factors[64];                  // 64 parts at most
  __shared__ float4 sums[kMergeThreads];
  __shared__ float all;
  const int parts = p.prefix_parts + p.own_parts, quads = p.head_dim / 4, slots = kMergeThreads / quads;
  const int slot = threadIdx.x / quads, quad = threadIdx.x - slot * quads;
  const long long pair = blockIdx.x, row = pair / p.q_heads;
  grid_dependency_wait();
  if (row < max(0, p.seq_starts[0]) || row >= min(p.rows, p.seq_starts[p.entries])) return;
  const float4* part_o = reinterpret_cast<const float4*>(p.part_o) + pair * parts * quads + quad;
  auto load = [&](int c) { return slot < slots && c < parts ? part_o[(size_t)c * quads] : make_float4(0.0f, 0.0f, 0.0f, 0.0f); };
  float4 first[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) first[i] = load(slot + i * slots);
  if (threadIdx.x < 32) {
    float2 ml[2];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = threadIdx.x + 32 * i;
      ml[i] = c < parts ? p.part_ml[pair * parts + c] : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, ml[i].x);
    }
    m = warp_max(m);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float factor = ml[i].x == -INFINITY ? (ml[i].y == 0.0f ? 0.0f : 1.0f) : exp2f(ml[i].x - m);   // (a part of nothing but NaN keeps its NaN)
      if (factor != 0.0f) l = fmaf(factor, ml[i].y, l);
      factors[threadIdx.x + 32 * i] = factor;
    }
    l = warp_sum(l);
    if (threadIdx.x == 0) all = l;
  }
  __syncthreads();
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (slot + i * slots < parts) add4(acc, factors[slot + i * slots], first[i]);
  for (int c = slot + 4 * slots; c < parts; c += 4 * slots) {
    float4 next[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) next[i] = load(c + i * slots);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i * slots < parts) add4(acc, factors[c + i * slots], next[i]);
  }
  sums[threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.x < quads) {
    for (int i = 1; i < slots; ++i) add4(acc, 1.0f, sums[i * quads + threadIdx.x]);
    T* out = (T*)p.out + (size_t)pair * p.head_dim + 4 * threadIdx.x;
    const float l = all;
    out[0] = from_float<T>(l == 0.0f ? 0.0f : acc.x / l), out[1] = from_float<T>(l == 0.0f ? 0.0f : acc.y / l);
    out[2] = from_float<T>(l == 0.0f ? 0.0f : acc.z / l), out[3] = from_float<T>(l == 0.0f ? 0.0f : acc.w / l);
  }
}

template <typename T, int MAX_DIM>
static int launch_generic(const SharedPrefixParams& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> devices{0};
  auto bytes = [](int dim) { return (int)sizeof(float) * (kPairs * (dim + 4) + kPairs * (kChunk + 4) + 2 * (kChunk * (dim + 4) + kChunk * dim)); };
  cudaError_t e = allow_shared_memory(shared_prefix_generic_kernel<T, MAX_DIM>, bytes(MAX_DIM), devices);
  if (e != cudaSuccess) return (int)e;
  const int group = p.q_heads / p.kv_heads;
  const long long tiles = ((long long)p.rows * group + kPairs - 1) / kPairs, ctas = tiles * p.prefix_parts + (tiles + p.entries) * p.own_parts;
  const long long pairs = (long long)p.rows * p.q_heads;
  if (ctas > 0x7fffffffLL || pairs > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  e = launch_pdl(shared_prefix_generic_kernel<T, MAX_DIM>, dim3((unsigned)ctas, p.kv_heads), dim3(kPairThreads), (size_t)bytes(p.head_dim), stream, p, (int)tiles);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(shared_prefix_merge_kernel<T>, dim3((unsigned)pairs), dim3(kMergeThreads), 0, stream, p);
}
template <typename T>
static int launch_generic(const SharedPrefixParams& p, cudaStream_t stream) {
  return p.head_dim <= 64 ? launch_generic<T, 64>(p, stream) : p.head_dim <= 128 ? launch_generic<T, 128>(p, stream) : launch_generic<T, 256>(p, stream);
}

}  // namespace tlie

using namespace tlie;

// q: rows [rows, q_row_stride] that start with the (rotated) query heads.  pages: one layer's pool [num_pages, 2, kv_heads, page_size, head_dim], 16-byte aligned.  out: [rows,
// q_heads * head_dim]; rows outside [seq_starts[0], seq_starts[entries]) are left as they are.  scratch: rows * q_heads * (prefix_parts + own_parts) *
// (head_dim + 2) floats, 16-byte aligned.
TLIE_EXPORT int tlie_shared_prefix_generic(int dtype, const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions, const int* seq_starts,
                                           const int* block_table, int table_stride, void* out, float* scratch, int rows, int entries, int q_heads, int kv_heads,
                                           int head_dim, int page_size, int shared, float scale, int prefix_parts, int own_parts, int* error_flag, cudaStream_t stream) {
  if (rows <= 0 || entries <= 0) return 0;
  if (head_dim <= 0 || head_dim > 256 || head_dim % 16 != 0 || kv_heads <= 0 || kv_heads > 65535 || q_heads % kv_heads != 0 || page_size <= 0 || num_pages <= 0 ||
      prefix_parts < 0 || own_parts < 1 || prefix_parts + own_parts > 64 || (prefix_parts == 0 && shared > 0) || error_flag == nullptr || ((uintptr_t)pages & 15) ||
      ((uintptr_t)scratch & 15))
    return (int)cudaErrorInvalidValue;
  const size_t parts = (size_t)rows * q_heads * (prefix_parts + own_parts);
  SharedPrefixParams p{q, q_row_stride, pages, num_pages, positions, seq_starts, block_table, table_stride, out, scratch, (float2*)(scratch + parts * head_dim),
                       rows, entries, q_heads, kv_heads, head_dim, page_size, shared, scale, prefix_parts, own_parts, error_flag};
  return dtype == TLIE_F32 ? launch_generic<float>(p, stream) : launch_generic<__nv_bfloat16>(p, stream);
}

extern "C" int tlie_prefix_tc(int, const void*, long long, const void*, int, const int*, const int*, const int*, int, void*, float*, float*, int, int, int, int, int, int, int, int, int, float,
                              int*, cudaStream_t);
extern "C" int tlie_prefix_rows(const void*, long long, const void*, int, const int*, const int*, const int*, int, void*, const float*, const float*, int, int, int, int, int, int, int, int,
                                float, int, int, int*, cudaStream_t);

// The bfloat16 kernels for head sizes 64 and 128 (each checks what it takes).  sizes, 13 numbers: prefix (0, every row reads the shared keys for itself; 1, the prefix's
// parts come from the tensor cores, `parts` runs of them), own (0, a row at a time, `ctas` per row and head; 1, an entry's rows on the tensor cores), parts, ctas, rows, entries, pages
// of a table row, q_heads, kv_heads, head_dim, page_size, shared, warps of those CTAs.  scratch: rows * q_heads * parts * (head_dim + 2) floats, 16-byte aligned.
TLIE_EXPORT int tlie_shared_prefix_bf16(const int* sizes, const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions, const int* seq_starts,
                                        const int* block_table, void* out, float* scratch, float scale, int* error_flag, cudaStream_t stream) {
  if (sizes == nullptr) return (int)cudaErrorInvalidValue;
  const int prefix = sizes[0], own = sizes[1], ctas = sizes[3], rows = sizes[4], entries = sizes[5], table_stride = sizes[6], q_heads = sizes[7], kv_heads = sizes[8];
  const int head_dim = sizes[9], page_size = sizes[10], shared = sizes[11];
  int parts = sizes[2];
  float *part_o = nullptr, *part_ml = nullptr;
  int first_key = 0, status = 0;
  if (prefix != 0) {
    if (scratch == nullptr) return (int)cudaErrorInvalidValue;
    part_o = scratch;
    part_ml = scratch + (size_t)rows * q_heads * parts * head_dim;
    first_key = shared;
    status = tlie_prefix_tc(0, q, q_row_stride, pages, num_pages, positions, seq_starts, block_table, table_stride, out, part_ml, part_o, parts, rows, entries, q_heads, kv_heads,
                            head_dim, page_size, shared, 0, scale, error_flag, stream);
    if (status != 0) return status;
  } else {
    parts = 0;
  }
  return own == 0 ? tlie_prefix_rows(q, q_row_stride, pages, num_pages, positions, seq_starts, block_table, table_stride, out, part_ml, part_o, parts, rows, entries, q_heads, kv_heads,
                                     head_dim, page_size, first_key, scale, ctas, sizes[12], error_flag, stream)
                  : tlie_prefix_tc(1, q, q_row_stride, pages, num_pages, positions, seq_starts, block_table, table_stride, out, part_ml, part_o, parts, rows, entries, q_heads, kv_heads,
                                   head_dim, page_size, shared, first_key, scale, error_flag, stream);
}
