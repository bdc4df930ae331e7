// Paged grouped-query attention of single query rows from a given key on, for batches whose requests share their first cached keys (bfloat16, head size 64 or
// 128, pages of a multiple of 16 keys): what attention_shared_prefix.cu computes, for steps of one decoded token per request.
//
// A cluster of CTAs owns one row, one key/value head and up to 16 of its query heads.  Its warps take the row's keys first_key <= j <= p 32 at a time, in turn;
// each keeps (m, l, o), the largest score, the sum of weights e^(s - m) and the weighted sum of values, of the keys it took.  At the end these parts are brought
// together with those that another kernel left for the keys below first_key, if there are any: with M the largest m, out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
//
// The bound is bytes: every key and value is read once and meets 16 query heads at most, in mma.sync of 16 x 8 x 16 (half of whose rows stand empty for groups of
// up to 8).  Keys and values go from global memory straight to the registers that the products read, 16 bytes a load, nothing in shared memory: which of
// a head's dims a product's k (or n) index stands for is free, as long as the query (or the output) agrees, so the four lanes of a key read 64 consecutive bytes of
// it, and the eight lanes that hold a value's n index 128.  A warp has a whole tile, 8 KB at head size 64 and 16 KB at 128, on its way at once.
#include <cooperative_groups.h>

#include "common.cuh"
#include "mma_utils.cuh"

namespace tlie {

constexpr int kRowWarps = 4;
constexpr int kRowHeads = 16;      // query heads of a CTA: the rows of a product
constexpr int kRowKeys = 32;       // keys of a tile
constexpr float kToLog2 = 1.4426950408889634f;
constexpr int kBadPage = 8;        // the bit of the device's error word

struct PrefixRowsParams {
  const __nv_bfloat16* q;
  long long q_row_stride;
  const __nv_bfloat16* pages;
  int num_pages;
  const int* positions;
  const int* seq_starts;
  const int* block_table;
  int table_stride;
  __nv_bfloat16* out;
  const float* part_o;      // [rows, q heads, parts, head size], the keys below first_key (null: none of them)
  const float2* part_ml;    // [rows, q heads, parts]: largest score in units of log2, sum of weights
  int parts, rows, entries, q_heads, kv_heads, page_size, first_key;
  float scale;
  int* error_flag;
};

__device__ __forceinline__ uint4 load_16(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }

// The entry that row t belongs to, -1 if it belongs to none.  In a step of one row per entry that is t itself.
__device__ __forceinline__ int entry_of_row(const int* seq_starts, int entries, int t) {
  if (t < entries && seq_starts[t] == t && seq_starts[t + 1] == t + 1) return t;
  int low = 0, high = entries;   // the last entry with seq_starts <= t
  if (t < seq_starts[0] || t >= seq_starts[entries]) return -1;
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (seq_starts[middle] <= t) low = middle;
    else high = middle;
  }
  return low;
}

template <int D>
__global__ void __launch_bounds__(kRowWarps * 32) prefix_rows_kernel(PrefixRowsParams p, bool waits_late) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row = blockIdx.x / ctas;
  const int group = p.q_heads / p.kv_heads, chunks = (group + kRowHeads - 1) / kRowHeads;
  const int kvh = blockIdx.y / chunks, head_in_group = (blockIdx.y - kvh * chunks) * kRowHeads;
  const int heads = min(kRowHeads, group - head_in_group), head0 = kvh * group + head_in_group;
  constexpr int kOutRow = D + 4;
  __shared__ __align__(16) float merge_o[kRowWarps][kRowHeads][kOutRow];
  __shared__ float2 merge_ml[kRowWarps][kRowHeads];
  __shared__ float weight_of[kRowWarps][kRowHeads];

  // The kernel in front may be the one that works out the parts of the keys below first_key.  It lets this one start when all its CTAs have waited for what came
  // before them; only its parts have to be waited for, at the end.
  if (!waits_late) grid_dependency_wait();

  const int entry = entry_of_row(p.seq_starts, p.entries, row);
  const long long room = (long long)p.table_stride * p.page_size;
  int limit = 0;
  if (entry >= 0) {
    long long seen = (long long)p.positions[row] + 1;
    if (seen > room) {
      if (threadIdx.x == 0) atomicOr(p.error_flag, kBadPage);
      seen = room;
    }
    limit = (int)max(seen, 0ll);
  }
  const int* table = p.block_table + (size_t)max(entry, 0) * p.table_stride;

  // this lane's part of q: for every 32 dims, 8 consecutive ones are what k = 2t, 2t + 1, 2t + 8, 2t + 9 of two products stand for
  unsigned qa[D / 16][4];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const __nv_bfloat16* q = p.q + (size_t)row * p.q_row_stride + (size_t)head0 * D + i * 32 + t * 8;
    uint4 low = make_uint4(0, 0, 0, 0), high = low;
    if (g < heads) low = load_16(q + (size_t)g * D);
    if (g + 8 < heads) high = load_16(q + (size_t)(g + 8) * D);
    qa[2 * i][0] = low.x, qa[2 * i][1] = high.x, qa[2 * i][2] = low.y, qa[2 * i][3] = high.y;
    qa[2 * i + 1][0] = low.z, qa[2 * i + 1][1] = high.z, qa[2 * i + 1][2] = low.w, qa[2 * i + 1][3] = high.w;
  }
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  const float to_log2 = p.scale * kToLog2;
  const bool upper = heads > 8;

  const int first_tile = p.first_key / kRowKeys, end_tile = (limit + kRowKeys - 1) / kRowKeys, step = ctas * kRowWarps;
  const size_t plane = (size_t)p.kv_heads * p.page_size * D;
  // Where the two halves of 16 keys of a tile start (each lies in one page).  What lies outside the table or the pool is reported, and page 0 read in its place.
  auto half_starts = [&](int tile, const __nv_bfloat16* (&start)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = tile * kRowKeys + 16 * h, index = key / p.page_size;
      int page = 0;
      if (key < limit) {
        page = table[index];
        if ((unsigned)page >= (unsigned)p.num_pages) {
          if (lane == 0) atomicOr(p.error_flag, kBadPage);
          page = 0;
        }
      }
      start[h] = p.pages + (size_t)page * 2 * plane + ((size_t)kvh * p.page_size + (key - index * p.page_size)) * D;
    }
  };
  int tile = first_tile + rank * kRowWarps + warp;
  const __nv_bfloat16* start[2];
  if (tile < end_tile) half_starts(tile, start);
  for (; tile < end_tile; tile += step) {
    const int key0 = tile * kRowKeys;
    const bool whole = key0 >= p.first_key && key0 + kRowKeys <= limit;
    uint4 k[4][D / 32], v[2][4][D / 64];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const __nv_bfloat16* key = start[n >> 1] + ((n & 1) * 8 + g) * D + t * 8;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) k[n][i] = load_16(key + i * 32);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int in_half = 2 * t + (r & 1) + (r >> 1) * 8, key = key0 + 16 * s + in_half;
        const __nv_bfloat16* value = start[s] + plane + in_half * D + g * 8;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) v[s][r][h] = whole || (key >= p.first_key && key < limit) ? load_16(value + h * 64) : make_uint4(0, 0, 0, 0);
      }
    if (tile + step < end_tile) half_starts(tile + step, start);

    float s[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        mma_bf16(s[n], qa[2 * i], k[n][i].x, k[n][i].y);
        mma_bf16(s[n], qa[2 * i + 1], k[n][i].z, k[n][i].w);
      }
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * n + 2 * t + (e & 1);
          if (key < p.first_key || key >= limit) s[n][e] = -INFINITY;
        }
    }
    float base[2], shrink[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float here = -INFINITY;
      if (r == 0 || upper) {
#pragma unroll
        for (int n = 0; n < 4; ++n) here = fmaxf(here, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
        here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 1));
        here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 2));
      }
      const float reference = fmaxf(top[r], here * to_log2);
      base[r] = reference == -INFINITY ? 0.0f : reference;
      shrink[r] = exp2_approx(top[r] - base[r]);
      top[r] = reference;
    }
    unsigned pa[2][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float p0 = exp2_approx(fmaf(s[n][0], to_log2, -base[0])), p1 = exp2_approx(fmaf(s[n][1], to_log2, -base[0]));
      if (n == 0) sum[0] *= shrink[0];
      sum[0] += p0 + p1;
      pa[n >> 1][(n & 1) * 2] = pack_bf16(p0, p1);   // a weight keeps 8 bits where it meets its value, as in the other bfloat16 attention kernels
      pa[n >> 1][(n & 1) * 2 + 1] = 0u;
    }
    if (upper) {
      sum[1] *= shrink[1];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float p0 = exp2_approx(fmaf(s[n][2], to_log2, -base[1])), p1 = exp2_approx(fmaf(s[n][3], to_log2, -base[1]));
        sum[1] += p0 + p1;
        pa[n >> 1][(n & 1) * 2 + 1] = pack_bf16(p0, p1);
      }
    }
    if (__any_sync(0xffffffffu, shrink[0] != 1.0f || shrink[1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] *= shrink[0], o[i][1] *= shrink[0], o[i][2] *= shrink[1], o[i][3] *= shrink[1];
    }
    // n index of product (h, i): dim h 64 + 8 n + i
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        const unsigned* r0 = &v[c][0][h].x;
        const unsigned* r1 = &v[c][1][h].x;
        const unsigned* r2 = &v[c][2][h].x;
        const unsigned* r3 = &v[c][3][h].x;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          mma_bf16(o[h * 8 + 2 * w], pa[c], __byte_perm(r0[w], r1[w], 0x5410), __byte_perm(r2[w], r3[w], 0x5410));
          mma_bf16(o[h * 8 + 2 * w + 1], pa[c], __byte_perm(r0[w], r1[w], 0x7632), __byte_perm(r2[w], r3[w], 0x7632));
        }
      }
  }

  // the warps' parts into shared memory
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    if (t == 0) merge_ml[warp][g + 8 * r] = make_float2(top[r], sum[r]);
    if (g + 8 * r < heads) {
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float* to = &merge_o[warp][g + 8 * r][h * 64 + (2 * t + half) * 8];
          const int e = 2 * r + half;
          *reinterpret_cast<float4*>(to) = make_float4(o[h * 8][e], o[h * 8 + 1][e], o[h * 8 + 2][e], o[h * 8 + 3][e]);
          *reinterpret_cast<float4*>(to + 4) = make_float4(o[h * 8 + 4][e], o[h * 8 + 5][e], o[h * 8 + 6][e], o[h * 8 + 7][e]);
        }
    }
  }
  __syncthreads();
  // this CTA's part into the place of its first warp's
  float2 mine[kRowWarps];
  for (int i = threadIdx.x; i < heads; i += blockDim.x) {
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      mine[w] = merge_ml[w][i];
      m = fmaxf(m, mine[w].x);
    }
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = mine[w].x == -INFINITY ? (mine[w].y == 0.0f ? 0.0f : 1.0f) : exp2f(mine[w].x - m);   // (a part of nothing but NaN keeps its NaN)
      weight_of[w][i] = f;
      l = fmaf(f, mine[w].y, l);
    }
    merge_ml[0][i] = make_float2(m, l);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (D / 4); i += blockDim.x) {
    const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = weight_of[w][h];
      if (f == 0.0f) continue;
      const float4 part = *reinterpret_cast<const float4*>(&merge_o[w][h][d]);
      acc.x = fmaf(f, part.x, acc.x), acc.y = fmaf(f, part.y, acc.y), acc.z = fmaf(f, part.z, acc.z), acc.w = fmaf(f, part.w, acc.w);
    }
    *reinterpret_cast<float4*>(&merge_o[0][h][d]) = acc;
  }
  if (ctas > 1) cluster.sync();
  else __syncthreads();
  if (waits_late) grid_dependency_wait();
  // the CTAs' parts and the ones of the keys below first_key: every CTA finishes its share of the output
  if (entry >= 0) {
    for (int i = rank * blockDim.x + threadIdx.x; i < heads * (D / 4); i += ctas * blockDim.x) {
      const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
      const size_t pair = (size_t)row * p.q_heads + head0 + h;
      float m = -INFINITY;
      for (int c = 0; c < ctas; ++c) m = fmaxf(m, cluster.map_shared_rank(&merge_ml[0][h], c)->x);
      for (int c = 0; c < p.parts; ++c) m = fmaxf(m, __ldcg(&p.part_ml[pair * p.parts + c]).x);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
      auto add = [&](float2 ml, const float4* part, bool global) {
        const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2f(ml.x - m);
        if (f == 0.0f) return;
        const float4 v = global ? __ldcg(part) : *part;
        l = fmaf(f, ml.y, l);
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
      };
      for (int c = 0; c < ctas; ++c)
        add(*cluster.map_shared_rank(&merge_ml[0][h], c), reinterpret_cast<const float4*>(cluster.map_shared_rank(&merge_o[0][h][d], c)), false);
      for (int c = 0; c < p.parts; ++c)
        add(__ldcg(&p.part_ml[pair * p.parts + c]), reinterpret_cast<const float4*>(p.part_o + (pair * p.parts + c) * D + d), true);
      const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
      uint2 packed = make_uint2(pack_bf16(acc.x * inverse, acc.y * inverse), pack_bf16(acc.z * inverse, acc.w * inverse));
      *reinterpret_cast<uint2*>(p.out + pair * D + d) = packed;
    }
  }
  if (ctas > 1) cluster.sync();   // a CTA's shared memory stays until the others have read it
}

template <int D>
static int launch_rows(const PrefixRowsParams& p, int ctas, bool waits_late, cudaStream_t stream) {
  const int group = p.q_heads / p.kv_heads, chunks = (group + kRowHeads - 1) / kRowHeads;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)p.rows * ctas, p.kv_heads * chunks);
  config.blockDim = dim3(kRowWarps * 32);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = ctas;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&config, prefix_rows_kernel<D>, p, waits_late);
}

}  // namespace tlie

using namespace tlie;

// q: rows [rows, q_row_stride] that start with the (rotated) query heads.  pages: one layer's pool [num_pages, 2, kv_heads, page_size, head_dim].  out: [rows,
// q_heads * head_dim]; rows outside [seq_starts[0], seq_starts[entries]) are left as they are.  ctas: 1, 2, 4 or 8 per (row, head).  parts: for every (row, query
// head), of the keys below first_key (0 if first_key is): 32-bit numbers [rows, q_heads, parts, 2] and then [rows, q_heads, parts, head_dim], 16-byte aligned
// from first to last.  With parts the kernel in front in the stream must be the one that writes them.
TLIE_EXPORT int tlie_prefix_rows(const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions, const int* seq_starts, const int* block_table,
                                 int table_stride, void* out, const float* part_ml, const float* part_o, int parts, int rows, int entries, int q_heads, int kv_heads,
                                 int head_dim, int page_size, int first_key, float scale, int ctas, int* error_flag, cudaStream_t stream) {
  if (rows <= 0 || entries <= 0) return 0;
  if (kv_heads <= 0 || q_heads % kv_heads != 0 || page_size <= 0 || page_size % 16 != 0 || num_pages <= 0 || q_row_stride % 8 != 0 || ((uintptr_t)q & 15) || ((uintptr_t)pages & 15) ||
      ((uintptr_t)out & 7) || ((uintptr_t)part_o & 15) || ((uintptr_t)part_ml & 7) || (ctas != 1 && ctas != 2 && ctas != 4 && ctas != 8) || (long long)rows * ctas > 0x7fffffffLL ||
      (long long)kv_heads * ((q_heads / kv_heads + kRowHeads - 1) / kRowHeads) > 65535 || error_flag == nullptr || (head_dim != 64 && head_dim != 128))
    return (int)cudaErrorInvalidValue;
  PrefixRowsParams p{(const __nv_bfloat16*)q, q_row_stride, (const __nv_bfloat16*)pages, num_pages, positions, seq_starts, block_table, table_stride, (__nv_bfloat16*)out,
                     part_o, (const float2*)part_ml, parts, rows, entries, q_heads, kv_heads, page_size, first_key, scale, error_flag};
  return head_dim == 64 ? launch_rows<64>(p, ctas, parts > 0, stream) : launch_rows<128>(p, ctas, parts > 0, stream);
}
