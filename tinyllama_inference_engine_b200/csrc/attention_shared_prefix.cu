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
// A CTA owns one key/value head, 32 (row, head) pairs and a run of keys, which it copies to shared memory 32 at a time: in a score a lane owns a key, in a
// weighted sum some of the value's channels.  All sums are 32-bit.
#include "common.cuh"
#include "shared_memory_limit.cuh"

namespace tlie {

constexpr int kPairs = 32;         // (row, head) pairs of a CTA
constexpr int kPairWarps = 4;
constexpr int kPairsPerWarp = kPairs / kPairWarps;
constexpr int kChunk = 32;         // keys in shared memory at a time: one per lane
constexpr int kDimsPerLane = 8;    // up to 256
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

template <typename T>
__global__ void __launch_bounds__(kPairWarps * 32) shared_prefix_generic_kernel(SharedPrefixParams p, int own_tiles) {
  extern __shared__ float smem[];
  const int D = p.head_dim, key_row = D + 4;   // four floats more: eight lanes that read 16 bytes of their keys' rows touch all banks
  float* q_smem = smem;                        // [pairs][D]
  float* k_smem = q_smem + kPairs * D;         // [keys][D + 4]
  float* v_smem = k_smem + kChunk * key_row;   // [keys][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, group = p.q_heads / p.kv_heads;
  const int first_row = max(0, p.seq_starts[0]), end_row = min(p.seq_starts[p.entries], p.rows);
  const bool of_prefix = (int)blockIdx.z < p.prefix_parts;
  const int part = blockIdx.z;

  // which pairs: consecutive ones of all rows, or of one entry's rows
  int row0, pairs, entry = 0;
  if (of_prefix) {
    const long long all = (long long)(end_row - first_row) * group, at = (long long)blockIdx.x * kPairs;
    if (at >= all) return;
    row0 = first_row;
    pairs = (int)min((long long)kPairs, all - at);
  } else {
    if ((int)blockIdx.x >= own_tiles) return;
    row0 = 0;
    pairs = 0;
  }
  long long pair0 = (long long)blockIdx.x * kPairs;
  if (!of_prefix) {   // the entry that this tile number falls to, counting every entry's tiles: 32 entries at a time
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
      const unsigned past = __ballot_sync(0xffffffffu, tiles_before + upto > (int)blockIdx.x);
      if (past != 0u) {
        const int at = __ffs(past) - 1;
        entry = e0 + at;
        const int before = tiles_before + __shfl_sync(0xffffffffu, upto - tiles, at);
        row0 = __shfl_sync(0xffffffffu, begin, at);
        const int rows_here = __shfl_sync(0xffffffffu, end, at) - row0;
        pair0 = (long long)((int)blockIdx.x - before) * kPairs;
        pairs = (int)min((long long)kPairs, (long long)rows_here * group - pair0);
        break;
      }
      tiles_before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (pairs <= 0) return;
  }
  // pair i of the tile: row and head
  auto row_of = [&](int i) { return row0 + (int)((pair0 + i) / group); };
  auto head_of = [&](int i) { return kvh * group + (int)((pair0 + i) % group); };

  const int* table = p.block_table + (size_t)entry * p.table_stride;
  const long long room = (long long)p.table_stride * p.page_size;
  // keys a pair sees in this kind of part: below `limit`
  auto limit_of = [&](int i) {
    long long seen = (long long)p.positions[row_of(i)] + 1;
    if (seen > room) {
      atomicOr(p.error_flag, kBadPage);
      seen = room;
    }
    return (int)(of_prefix ? min(seen, (long long)p.shared) : seen);
  };
  int last = 0;
  for (int i = lane; i < pairs; i += 32) last = max(last, limit_of(i));
  last = __reduce_max_sync(0xffffffffu, last);
  const int from = of_prefix ? 0 : p.shared;
  const int chunks = last > from ? (last - from + kChunk - 1) / kChunk : 0;
  const int parts_here = of_prefix ? p.prefix_parts : p.own_parts, which = of_prefix ? part : part - p.prefix_parts;
  const int per_part = (chunks + parts_here - 1) / parts_here;
  const int chunk_begin = which * per_part, chunk_end = min(chunks, chunk_begin + per_part);

  for (int i = threadIdx.x; i < kPairs * D; i += blockDim.x) {
    const int pair = i / D, d = i - pair * D;
    q_smem[i] = pair < pairs ? to_float(((const T*)p.q)[(size_t)row_of(pair) * p.q_row_stride + (size_t)head_of(pair) * D + d]) * p.scale * kToLog2 : 0.0f;
  }
  int limit[kPairsPerWarp];
  float top[kPairsPerWarp], sum[kPairsPerWarp], acc[kPairsPerWarp][kDimsPerLane];
#pragma unroll
  for (int r = 0; r < kPairsPerWarp; ++r) {
    const int i = warp * kPairsPerWarp + r;
    limit[r] = i < pairs ? limit_of(i) : 0;
    top[r] = -INFINITY;
    sum[r] = 0.0f;
#pragma unroll
    for (int c = 0; c < kDimsPerLane; ++c) acc[r][c] = 0.0f;
  }
  const size_t plane = (size_t)p.kv_heads * p.page_size * D;
  for (int chunk = chunk_begin; chunk < chunk_end; ++chunk) {
    const int key0 = from + chunk * kChunk, keys = min(kChunk, last - key0);
    __syncthreads();
    for (int j = warp; j < kChunk; j += kPairWarps) {
      if (j < keys) {
        const int key = key0 + j, page = page_of(p, table, key / p.page_size);
        const T* k_row = (const T*)p.pages + (size_t)page * 2 * plane + ((size_t)kvh * p.page_size + key % p.page_size) * D;
        for (int d = lane; d < D; d += 32) {
          k_smem[j * key_row + d] = to_float(k_row[d]);
          v_smem[j * D + d] = to_float(k_row[plane + d]);
        }
      } else {
        for (int d = lane; d < D; d += 32) k_smem[j * key_row + d] = v_smem[j * D + d] = 0.0f;
      }
    }
    __syncthreads();
    float score[kPairsPerWarp];
#pragma unroll
    for (int r = 0; r < kPairsPerWarp; ++r) score[r] = 0.0f;
    for (int d = 0; d < D; d += 4) {
      const float4 k4 = *reinterpret_cast<const float4*>(k_smem + lane * key_row + d);
#pragma unroll
      for (int r = 0; r < kPairsPerWarp; ++r) {
        const float4 q4 = *reinterpret_cast<const float4*>(q_smem + (warp * kPairsPerWarp + r) * D + d);
        score[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, score[r]))));
      }
    }
#pragma unroll
    for (int r = 0; r < kPairsPerWarp; ++r) {
      const bool seen = key0 + lane < limit[r];
      const float s = seen ? score[r] : -INFINITY;
      const float reference = fmaxf(top[r], warp_max(s));
      const float base = reference == -INFINITY ? 0.0f : reference;
      const float shrink = top[r] == -INFINITY ? 0.0f : exp2f(top[r] - base);
      const float w = seen ? exp2f(s - base) : 0.0f;
      top[r] = reference;
      sum[r] = fmaf(sum[r], shrink, warp_sum(w));
#pragma unroll
      for (int c = 0; c < kDimsPerLane; ++c) acc[r][c] *= shrink;
      score[r] = w;
    }
    // Only keys that a pair sees are added: what lies in another's later places (it may be no number) must not reach it through a weight of zero.
#pragma unroll
    for (int r = 0; r < kPairsPerWarp; ++r) {
      const int seen = min(keys, limit[r] - key0);
      for (int j = 0; j < seen; ++j) {
        const float w = __shfl_sync(0xffffffffu, score[r], j);
#pragma unroll
        for (int c = 0; c < kDimsPerLane; ++c)
          if (lane + 32 * c < D) acc[r][c] = fmaf(w, v_smem[j * D + lane + 32 * c], acc[r][c]);
      }
    }
  }
  const int parts = p.prefix_parts + p.own_parts;
#pragma unroll
  for (int r = 0; r < kPairsPerWarp; ++r) {
    const int i = warp * kPairsPerWarp + r;
    if (i >= pairs) break;
    const size_t at = ((size_t)row_of(i) * p.q_heads + head_of(i)) * parts + part;
    if (lane == 0) p.part_ml[at] = make_float2(top[r], sum[r]);
#pragma unroll
    for (int c = 0; c < kDimsPerLane; ++c)
      if (lane + 32 * c < D) p.part_o[at * D + lane + 32 * c] = acc[r][c];
  }
}

// One warp per (row, head): the parts brought together.  A row that sees no key gives zeros.
template <typename T>
__global__ void shared_prefix_merge_kernel(SharedPrefixParams p) {
  const int lane = threadIdx.x & 31, parts = p.prefix_parts + p.own_parts, D = p.head_dim;
  const long long pair = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const long long row = pair / p.q_heads;
  if (row < max(0, p.seq_starts[0]) || row >= min(p.rows, p.seq_starts[p.entries])) return;
  const float2* ml = p.part_ml + pair * parts;
  float top = -INFINITY;
  for (int i = 0; i < parts; ++i) top = fmaxf(top, ml[i].x);
  float acc[kDimsPerLane] = {0.0f}, sum = 0.0f;
  for (int i = 0; i < parts; ++i) {
    const float2 here = ml[i];
    const float factor = here.x == -INFINITY ? 0.0f : exp2f(here.x - top);
    if (here.y == 0.0f) continue;
    sum = fmaf(factor, here.y, sum);
#pragma unroll
    for (int c = 0; c < kDimsPerLane; ++c)
      if (lane + 32 * c < D) acc[c] = fmaf(factor, p.part_o[((size_t)pair * parts + i) * D + lane + 32 * c], acc[c]);
  }
#pragma unroll
  for (int c = 0; c < kDimsPerLane; ++c)
    if (lane + 32 * c < D) ((T*)p.out)[(size_t)pair * D + lane + 32 * c] = from_float<T>(sum == 0.0f ? 0.0f : acc[c] / sum);
}

template <typename T>
static int launch_generic(const SharedPrefixParams& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> devices{0};
  const size_t smem = sizeof(float) * (size_t)(kPairs * p.head_dim + kChunk * (p.head_dim + 4) + kChunk * p.head_dim);
  cudaError_t e = allow_shared_memory(shared_prefix_generic_kernel<T>, (int)(sizeof(float) * (kPairs * 256 + kChunk * 260 + kChunk * 256)), devices);
  if (e != cudaSuccess) return (int)e;
  const int group = p.q_heads / p.kv_heads;
  const long long tiles = ((long long)p.rows * group + kPairs - 1) / kPairs, own_tiles = tiles + p.entries;
  const long long pairs = (long long)p.rows * p.q_heads;
  if (own_tiles > 0x7fffffffLL || (pairs + 7) / 8 > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  shared_prefix_generic_kernel<T><<<dim3((unsigned)own_tiles, p.kv_heads, p.prefix_parts + p.own_parts), kPairWarps * 32, smem, stream>>>(p, (int)own_tiles);
  e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  shared_prefix_merge_kernel<T><<<(unsigned)((pairs + 7) / 8), 256, 0, stream>>>(p);
  return (int)cudaGetLastError();
}

}  // namespace tlie

using namespace tlie;

// q: rows [rows, q_row_stride] that start with the (rotated) query heads.  pages: one layer's pool [num_pages, 2, kv_heads, page_size, head_dim].  out: [rows,
// q_heads * head_dim]; rows outside [seq_starts[0], seq_starts[entries]) are left as they are.  scratch: rows * q_heads * (prefix_parts + own_parts) *
// (head_dim + 2) floats, 8-byte aligned.
TLIE_EXPORT int tlie_shared_prefix_generic(int dtype, const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions, const int* seq_starts,
                                           const int* block_table, int table_stride, void* out, float* scratch, int rows, int entries, int q_heads, int kv_heads,
                                           int head_dim, int page_size, int shared, float scale, int prefix_parts, int own_parts, int* error_flag, cudaStream_t stream) {
  if (rows <= 0 || entries <= 0) return 0;
  if (head_dim <= 0 || head_dim > 256 || head_dim % 4 != 0 || kv_heads <= 0 || kv_heads > 65535 || q_heads % kv_heads != 0 || page_size <= 0 || num_pages <= 0 ||
      prefix_parts < 0 || own_parts < 1 || prefix_parts + own_parts > 65535 || (prefix_parts == 0 && shared > 0) || error_flag == nullptr)
    return (int)cudaErrorInvalidValue;
  const size_t parts = (size_t)rows * q_heads * (prefix_parts + own_parts);
  SharedPrefixParams p{q, q_row_stride, pages, num_pages, positions, seq_starts, block_table, table_stride, out, scratch + 2 * parts, (float2*)scratch,
                       rows, entries, q_heads, kv_heads, head_dim, page_size, shared, scale, prefix_parts, own_parts, error_flag};
  return dtype == TLIE_F32 ? launch_generic<float>(p, stream) : launch_generic<__nv_bfloat16>(p, stream);
}

extern "C" int tlie_prefix_tc(int, const void*, long long, const void*, int, const int*, const int*, const int*, int, void*, float*, float*, int, int, int, int, int, int, int, int, int, float,
                              int*, cudaStream_t);
extern "C" int tlie_prefix_rows(const void*, long long, const void*, int, const int*, const int*, const int*, int, void*, const float*, const float*, int, int, int, int, int, int, int, int,
                                float, int, int*, cudaStream_t);

// The bfloat16 kernels for head sizes 64 and 128 (each checks what it takes).  prefix: 0, every row reads the shared keys for itself; 1, the prefix's parts come
// from the tensor cores, `parts` runs of them.  own: 0, a row at a time (`ctas` per row and head), 1, an entry's rows on the tensor cores.
// scratch: rows * q_heads * parts * (head_dim + 2) floats, 16-byte aligned.
TLIE_EXPORT int tlie_shared_prefix_bf16(int prefix, int own, int parts, int ctas, const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions,
                                        const int* seq_starts, const int* block_table, int table_stride, void* out, float* scratch, int rows, int entries, int q_heads, int kv_heads,
                                        int head_dim, int page_size, int shared, float scale, int* error_flag, cudaStream_t stream) {
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
                                     head_dim, page_size, first_key, scale, ctas, error_flag, stream)
                  : tlie_prefix_tc(1, q, q_row_stride, pages, num_pages, positions, seq_starts, block_table, table_stride, out, part_ml, part_o, parts, rows, entries, q_heads, kv_heads,
                                   head_dim, page_size, shared, first_key, scale, error_flag, stream);
}
