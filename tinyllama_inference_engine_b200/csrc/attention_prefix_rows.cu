// Paged grouped-query attention of single query rows from a given key on, for batches whose requests share their first cached keys (bfloat16, head size 64 or
// 128, pages of a multiple of 16 keys): what attention_shared_prefix.cu computes, for steps of one decoded token per request.
//
// A cluster of CTAs owns one row, one key/value head and up to 8 of its query heads.  Its warps take the row's keys first_key <= j <= p 16 at a time, in turn;
// each keeps (m, l, o), the largest score, the sum of weights e^(s - m) and the weighted sum of values, of the keys it took.  At the end these parts are brought
// together with those that another kernel left for the keys below first_key, if there are any: with M the largest m, out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
//
// The bound is bytes: every key and value is read once and meets 8 query heads at most.  Both products are mma.sync of 16 x 8 x 16 with the keys, or the values' dims, as the 16
// rows and the query heads as the 8 columns (heads as rows would leave half of the rows of every product and half of the output's registers empty).  Keys and values go
// from global memory straight to the registers that the products read, 16 bytes a load, nothing in shared memory: which of a head's dims a product's k index, or a row of
// its output, stands for is free, as long as the query agrees, so the four lanes of a key read 64 consecutive bytes of it, and the eight lanes of a value 128.  A
// warp has a whole tile, 4 KB at head size 64 and 8 KB at 128, on its way at once.
//
// CTAs of few warps where there are many: a CTA's start and end (the chain from the table to its first key, its parts' joining) cost an SM more than the keys of a short request, and
// 16 warps are on an SM either way (128 registers a thread).  48 rows, 32 heads of 128, 612 keys each on average, behind 2,192 shared ones: 481 MB in 84 us beside the prefix's 17, 0.88 of the
// measured copy rate.  131 rows, 32 heads, 24 keys: 33 us with the prefix's 17 (8 warps: 73).  64 rows, 4 key/value heads of 64 for 8 query heads each, 870 keys: 11.9 us, 4.8 TB/s from L2; one row behind 305: 5 us.
#include <cooperative_groups.h>

#include <cstdlib>

#include "common.cuh"
#include "mma_utils.cuh"
#include "shared_memory_limit.cuh"

namespace tlie {

constexpr int kRowWarps = 16;      // at most
constexpr int kRowHeads = 8;       // query heads of a CTA: the columns of a product
constexpr int kRowKeys = 16;       // keys of a tile: the rows of a product
constexpr int kMostParts = 64;     // of the keys below first_key
constexpr int kMostSources = kRowWarps + kMostParts;   // (a CTA's warps, or a cluster's CTAs, and the parts)
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

// The entry that row t belongs to, -1 if it belongs to none.
__device__ __noinline__ int entry_of_row(const int* seq_starts, int entries, int t) {
  int low = 0, high = entries;   // the last entry with seq_starts <= t
  if (t < seq_starts[0] || t >= seq_starts[entries]) return -1;
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (seq_starts[middle] <= t) low = middle;
    else high = middle;
  }
  return low;
}

// Rows and columns of 8 x 8 16-bit numbers exchanged: lane (g, t) has numbers 2t, 2t + 1 of row g before, and of column g after.
__device__ __forceinline__ unsigned transpose_8x8(unsigned two) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(two));
  return r;
}

template <int D>
__global__ void __launch_bounds__(kRowWarps * 32, 1) prefix_rows_kernel(PrefixRowsParams p, bool waits_late) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank(), warps = blockDim.x >> 5;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row = blockIdx.x / ctas;
  const int group = p.q_heads / p.kv_heads, chunks = (group + kRowHeads - 1) / kRowHeads;
  const int kvh = blockIdx.y / chunks, head_in_group = (blockIdx.y - kvh * chunks) * kRowHeads;
  const int heads = min(kRowHeads, group - head_in_group), head0 = kvh * group + head_in_group;
  constexpr int kOutRow = D + 4;
  extern __shared__ __align__(16) float merge_o[];   // [warp][head][kOutRow]
  __shared__ float2 merge_ml[kRowWarps][kRowHeads];
  __shared__ float factor_of[kRowHeads][kMostSources];

  // The kernel in front may be the one that works out the parts of the keys below first_key.  It lets this one start when all its CTAs have waited for what came
  // before them; only its parts have to be waited for, at the end.
  if (!waits_late) grid_dependency_wait();

  // A step of one row per entry is asked for as such, all of it in one trip to memory; where the guess is wrong the entry is looked for.
  const int warp_in_row = rank * warps + warp, step = ctas * warps;
  int tile = p.first_key / kRowKeys + warp_in_row;
  int entry = min(row, p.entries - 1);
  auto table_page = [&](const int* table, int tile) {
    const int index = tile * kRowKeys / p.page_size;
    return index < p.table_stride ? table[index] : -1;
  };
  const int* table = p.block_table + (size_t)entry * p.table_stride;
  const int begins = p.seq_starts[entry], ends = p.seq_starts[entry + 1];
  long long seen = (long long)p.positions[row] + 1;
  int page = table_page(table, tile);
  if (begins != row || ends != row + 1) {
    entry = entry_of_row(p.seq_starts, p.entries, row);
    table = p.block_table + (size_t)max(entry, 0) * p.table_stride;
    page = table_page(table, tile);
  }
  const long long room = (long long)p.table_stride * p.page_size;
  int limit = 0;
  if (entry >= 0) {
    if (seen > room) {
      if (threadIdx.x == 0) atomicOr(p.error_flag, kBadPage);
      seen = room;
    }
    limit = (int)max(seen, 0ll);
  }

  // this lane's part of q, head g: for every 32 dims, 8 consecutive ones are what k = 2t, 2t + 1, 2t + 8, 2t + 9 of two products stand for
  uint4 q[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    q[i] = g < heads ? load_16(p.q + (size_t)row * p.q_row_stride + (size_t)(head0 + g) * D + i * 32 + t * 8) : make_uint4(0, 0, 0, 0);
  float o[D / 16][4];   // product (h, i): rows g and g + 8 are dims h 64 + 8 g + 2 i and the next, columns 2 t and 2 t + 1 the heads
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};   // of heads 2 t and 2 t + 1
  const float to_log2 = p.scale * kToLog2;
  const int end_tile = (limit + kRowKeys - 1) / kRowKeys;
  const size_t plane = (size_t)p.kv_heads * p.page_size * D;
  for (; tile < end_tile; tile += step) {
    const int key0 = tile * kRowKeys;   // (a tile lies in one page)
    if ((unsigned)page >= (unsigned)p.num_pages) {   // reported, and page 0 read in its place
      if (lane == 0) atomicOr(p.error_flag, kBadPage);
      page = 0;
    }
    const __nv_bfloat16* start = p.pages + (size_t)page * 2 * plane + ((size_t)kvh * p.page_size + key0 % p.page_size) * D;
    const bool whole = key0 >= p.first_key && key0 + kRowKeys <= limit;
    uint4 k[2][D / 32], v[4][D / 64];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) k[r][i] = load_16(start + (g + 8 * r) * D + t * 8 + i * 32);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int in_tile = 2 * t + (r & 1) + (r >> 1) * 8, key = key0 + in_tile;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        v[r][h] = whole || (key >= p.first_key && key < limit) ? load_16(start + plane + in_tile * D + g * 8 + h * 64) : make_uint4(0, 0, 0, 0);
    }
    page = table_page(table, tile + step);

    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // keys g (0, 1) and g + 8 (2, 3), heads 2 t and 2 t + 1
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const unsigned first[4] = {k[0][i].x, k[1][i].x, k[0][i].y, k[1][i].y}, second[4] = {k[0][i].z, k[1][i].z, k[0][i].w, k[1][i].w};
      mma_bf16(s, first, q[i].x, q[i].y);
      mma_bf16(s, second, q[i].z, q[i].w);
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + g + (e >> 1) * 8;
        if (key < p.first_key || key >= limit) s[e] = -INFINITY;
      }
    }
    float base[2], shrink[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float here = fmaxf(s[h], s[h + 2]);
#pragma unroll
      for (int other = 4; other < 32; other <<= 1) here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, other));
      const float reference = fmaxf(top[h], here * to_log2);
      base[h] = reference == -INFINITY ? 0.0f : reference;
      shrink[h] = exp2_approx(top[h] - base[h]);
      top[h] = reference;
    }
    const float p0 = exp2_approx(fmaf(s[0], to_log2, -base[0])), p1 = exp2_approx(fmaf(s[1], to_log2, -base[1]));
    const float p2 = exp2_approx(fmaf(s[2], to_log2, -base[0])), p3 = exp2_approx(fmaf(s[3], to_log2, -base[1]));
    sum[0] = fmaf(sum[0], shrink[0], p0 + p2);
    sum[1] = fmaf(sum[1], shrink[1], p1 + p3);
    // a weight keeps 8 bits where it meets its value, as in the other bfloat16 attention kernels (the product takes bfloat16): an error like that of the output's own rounding
    const unsigned w0 = transpose_8x8(pack_bf16(p0, p1)), w1 = transpose_8x8(pack_bf16(p2, p3));
    if (__any_sync(0xffffffffu, shrink[0] != 1.0f || shrink[1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i][0] *= shrink[0], o[i][1] *= shrink[1], o[i][2] *= shrink[0], o[i][3] *= shrink[1];
    }
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const unsigned* r0 = &v[0][h].x;
      const unsigned* r1 = &v[1][h].x;
      const unsigned* r2 = &v[2][h].x;
      const unsigned* r3 = &v[3][h].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned a[4] = {__byte_perm(r0[i], r1[i], 0x5410), __byte_perm(r0[i], r1[i], 0x7632), __byte_perm(r2[i], r3[i], 0x5410), __byte_perm(r2[i], r3[i], 0x7632)};
        mma_bf16(o[h * 4 + i], a, w0, w1);
      }
    }
  }

  // the warps' parts into shared memory
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int other = 4; other < 32; other <<= 1) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], other);
    if (g == 0) merge_ml[warp][2 * t + h] = make_float2(top[h], sum[h]);
    if (2 * t + h >= heads) continue;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      float* to = merge_o + (warp * heads + 2 * t + h) * kOutRow + b * 64 + g * 8;
      *reinterpret_cast<float4*>(to) = make_float4(o[b * 4][h], o[b * 4][h + 2], o[b * 4 + 1][h], o[b * 4 + 1][h + 2]);
      *reinterpret_cast<float4*>(to + 4) = make_float4(o[b * 4 + 2][h], o[b * 4 + 2][h + 2], o[b * 4 + 3][h], o[b * 4 + 3][h + 2]);
    }
  }
  __syncthreads();
  // Parts are weighed head by head: a warp each, the parts over its lanes; (m, l) of them all, and what each counts for in units of the largest.
  constexpr int kPerLane = (kMostSources + 31) / 32;
  auto weigh = [&](float2 (&ml)[kPerLane]) {
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) m = fmaxf(m, ml[i].x);
    m = warp_max(m);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      ml[i].x = ml[i].x == -INFINITY ? (ml[i].y == 0.0f ? 0.0f : 1.0f) : exp2f(ml[i].x - m);   // (a part of nothing but NaN keeps its NaN)
      if (ml[i].x != 0.0f) l = fmaf(ml[i].x, ml[i].y, l);
    }
    return make_float2(m, warp_sum(l));
  };
  if (ctas > 1) {   // this CTA's part into the place of its first warp's, for the cluster
    for (int h = warp; h < heads; h += warps) {
      float2 ml[kPerLane];
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) ml[i] = lane + 32 * i < warps ? merge_ml[lane + 32 * i][h] : make_float2(-INFINITY, 0.0f);
      const float2 together = weigh(ml);
      if (lane < warps) factor_of[h][lane] = ml[0].x;
      __syncwarp();
      if (lane == 0) merge_ml[0][h] = together;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (D / 4); i += blockDim.x) {
      const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
      for (int w = 0; w < warps; ++w) {
        const float f = factor_of[h][w];
        float4 part = *reinterpret_cast<const float4*>(merge_o + (w * heads + h) * kOutRow + d);
        if (f == 0.0f) part = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // (what counts for nothing may be no number)
        acc.x = fmaf(f, part.x, acc.x), acc.y = fmaf(f, part.y, acc.y), acc.z = fmaf(f, part.z, acc.z), acc.w = fmaf(f, part.w, acc.w);
      }
      *reinterpret_cast<float4*>(merge_o + h * kOutRow + d) = acc;
    }
    cluster.sync();
  }
  if (waits_late) grid_dependency_wait();

  // the cluster's CTAs' parts (or this CTA's warps') and those of the keys below first_key
  const int own_sources = ctas > 1 ? ctas : warps, sources = own_sources + p.parts;
  for (int h = warp; h < heads && entry >= 0; h += warps) {
    const size_t pair = (size_t)row * p.q_heads + head0 + h;
    float2 ml[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int source = lane + 32 * i;
      ml[i] = make_float2(-INFINITY, 0.0f);
      if (source < own_sources) ml[i] = ctas > 1 ? *cluster.map_shared_rank(&merge_ml[0][h], source) : merge_ml[source][h];
      else if (source < sources) ml[i] = __ldcg(&p.part_ml[pair * p.parts + source - own_sources]);
    }
    const float l = weigh(ml).y;
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < sources) factor_of[h][lane + 32 * i] = ml[i].x == 0.0f ? 0.0f : ml[i].x * inverse;
  }
  __syncthreads();
  // every CTA of the cluster finishes its share of the output; a part that counts for nothing is not read (it may never have been written)
  if (entry >= 0) {
    for (int i = rank * blockDim.x + threadIdx.x; i < heads * (D / 4); i += ctas * blockDim.x) {
      const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
      const size_t pair = (size_t)row * p.q_heads + head0 + h;
      const float* factor = factor_of[h];
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      auto add = [&](float f, float4 part) { acc.x = fmaf(f, part.x, acc.x), acc.y = fmaf(f, part.y, acc.y), acc.z = fmaf(f, part.z, acc.z), acc.w = fmaf(f, part.w, acc.w); };
      const float4 nothing = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int c = 0; c < p.parts; ++c) {
        const float f = factor[own_sources + c];
        add(f, f != 0.0f ? __ldcg(reinterpret_cast<const float4*>(p.part_o + (pair * p.parts + c) * D + d)) : nothing);
      }
#pragma unroll 4
      for (int c = 0; c < own_sources; ++c) {
        const float f = factor[c];
        const float* from = ctas > 1 ? cluster.map_shared_rank(merge_o + h * kOutRow + d, c) : merge_o + (c * heads + h) * kOutRow + d;
        add(f, f != 0.0f ? *reinterpret_cast<const float4*>(from) : nothing);
      }
      *reinterpret_cast<uint2*>(p.out + pair * D + d) = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
    }
  }
  if (ctas > 1) cluster.sync();   // a CTA's shared memory stays until the others have read it
}

template <int D>
static int launch_rows(const PrefixRowsParams& p, int ctas, int warps, bool waits_late, cudaStream_t stream) {
  static std::atomic<unsigned long long> devices{0};
  const cudaError_t e = allow_shared_memory(prefix_rows_kernel<D>, (int)sizeof(float) * kRowWarps * kRowHeads * (D + 4), devices);
  if (e != cudaSuccess) return (int)e;
  const int group = p.q_heads / p.kv_heads, chunks = (group + kRowHeads - 1) / kRowHeads;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)p.rows * ctas, p.kv_heads * chunks);
  config.blockDim = dim3(warps * 32);
  config.dynamicSmemBytes = sizeof(float) * warps * (group < kRowHeads ? group : kRowHeads) * (D + 4);
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
  return (int)cudaLaunchKernelEx(&config, prefix_rows_kernel<D>, p, waits_late);
}

}  // namespace tlie

using namespace tlie;

// q: rows [rows, q_row_stride] that start with the (rotated) query heads.  pages: one layer's pool [num_pages, 2, kv_heads, page_size, head_dim].  out: [rows,
// q_heads * head_dim]; rows outside [seq_starts[0], seq_starts[entries]) are left as they are.  ctas: 1, 2, 4 or 8 per (row, head), of 1 to 16 warps.  parts: for every (row, query
// head), of the keys below first_key (0 if first_key is): 32-bit numbers [rows, q_heads, parts, 2] and then [rows, q_heads, parts, head_dim], 16-byte aligned
// from first to last.  With parts the kernel in front in the stream must be the one that writes them.
TLIE_EXPORT int tlie_prefix_rows(const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions, const int* seq_starts, const int* block_table,
                                 int table_stride, void* out, const float* part_ml, const float* part_o, int parts, int rows, int entries, int q_heads, int kv_heads,
                                 int head_dim, int page_size, int first_key, float scale, int ctas, int warps, int* error_flag, cudaStream_t stream) {
  if (rows <= 0 || entries <= 0) return 0;
  if (kv_heads <= 0 || q_heads % kv_heads != 0 || page_size <= 0 || page_size % 16 != 0 || num_pages <= 0 || q_row_stride % 8 != 0 || ((uintptr_t)q & 15) || ((uintptr_t)pages & 15) ||
      ((uintptr_t)out & 7) || ((uintptr_t)part_o & 15) || ((uintptr_t)part_ml & 7) || parts < 0 || parts > kMostParts || (ctas != 1 && ctas != 2 && ctas != 4 && ctas != 8) || warps < 1 || warps > kRowWarps || (long long)rows * ctas > 0x7fffffffLL ||
      (long long)kv_heads * ((q_heads / kv_heads + kRowHeads - 1) / kRowHeads) > 65535 || error_flag == nullptr || (head_dim != 64 && head_dim != 128))
    return (int)cudaErrorInvalidValue;
  PrefixRowsParams p{(const __nv_bfloat16*)q, q_row_stride, (const __nv_bfloat16*)pages, num_pages, positions, seq_starts, block_table, table_stride, (__nv_bfloat16*)out,
                     part_o, (const float2*)part_ml, parts, rows, entries, q_heads, kv_heads, page_size, first_key, scale, error_flag};
  return head_dim == 64 ? launch_rows<64>(p, ctas, warps, parts > 0, stream) : launch_rows<128>(p, ctas, warps, parts > 0, stream);
}
