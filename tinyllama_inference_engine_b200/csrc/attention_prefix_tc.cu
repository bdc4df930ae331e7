// Paged grouped-query attention for batches whose requests share their first cached keys, on the 5th-generation tensor cores (bfloat16, head size 64 or 128,
// pages of a multiple of 16 keys).  Two builds of one kernel:
//   * of the prefix (OWN false): all rows of the step against the keys below `shared`, a run of which a CTA takes; it leaves (m, l, o) per (row, query head): the
//     largest score (a reference near it), the sum of weights and the weighted sum of values;
//   * of an entry's own keys (OWN true): an entry's rows against its keys first_key <= j <= p, brought together with the parts of the prefix where there are any,
//     to the finished output.  With first_key = 0 it is the whole attention of portions of many rows.
//
// The query heads of a group meet the same keys: a row tile is 128 (row, head of the group) pairs, 128 / group rows of the step.  A CTA has two such tiles and a
// ring of key and value tiles (128 keys) for both, so that keys and values come from L2 once per 256 pairs, and so that one tile's products run
// under the other's softmax: with 512 columns of tensor memory there is one score buffer and one output per tile (128 columns each), and what is in turn for a tile (scores, softmax,
// weighted values) alternates between the two.  One CTA fills an SM.
//   * TMA brings Q once (a box of 64 dims x the group's heads x 128 / group rows per half), and every key tile as boxes that lie inside a page.  The lanes of
//     the producing warp each look up one box's page and copy it;
//   * S = Q . K^T (128 x 128 x head size) and O += P . V (128 x head size x 128) are issued by one thread per row tile.  P lies in tensor memory, over the
//     first half of its scores, and is handed over in halves: the product of the first 64 keys runs under the exponentials of the others;
//   * thread = (row, head) pair = lane of tensor memory: maxima and sums need no other thread.  The output is taken against a reference maximum that
//     moves only when a tile's maximum is more than 2^8 above it;
//   * what a tile's rows do not all see is masked; a value that some of them see and that is not finite would spread through a weight of zero, so in such tiles values are looked
//     through, what is not finite is taken out and noted, and the rows that do see it show it in the end.
// Every wait is bounded; a CTA that gives up raises the device's error word, lets its copies land and returns.
#include "shared_memory_limit.cuh"
#include "tcgen05_utils.cuh"

namespace tlie {

constexpr int kPairsTC = 128;       // (row, head) pairs of a row tile
constexpr int kKeysTC = 128;        // keys of a key tile
constexpr int kBoxDims = 64;        // dims of one box: 128 bytes, the swizzle span
constexpr int kThreadsTC = 384;     // warps 0 copies, 1 and 2 products, 3 none, 4 to 7 and 8 to 11 softmax of the two row tiles
constexpr int kFirstSoftmaxWarp = 4;
constexpr int kControlRegs = 56, kSoftmaxRegs = 224, kLaunchRegs = 168;   // 128 * 56 + 256 * 224 = 384 * 168
constexpr float kToLog2 = 1.4426950408889634f;
constexpr float kLazyRescale = 8.0f;
constexpr int kBadPage = 8;         // the bit of the device's error word
constexpr int kNoKey = 0x7fffffff;

// bf16 x bf16 -> f32, A K-major, B MN-major (V stays [key][dim], as the cache stores it), tile m x n.
__host__ __device__ constexpr uint32_t instr_desc_b_mn(int m, int n) { return umma_instr_desc(m, n) | (1u << 16); }

__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
  uint32_t r[32], s[32];
  tmem_load_32(taddr, r);
  tmem_load_32(taddr + 32, s);
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]), v[32 + i] = __uint_as_float(s[i]);
}
__device__ __forceinline__ void tmem_store_32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
// The product with its A operand in tensor memory (lane = row, 16 k = 8 columns of two bfloat16) and B by its descriptor's lower word.
__device__ __forceinline__ void umma_bf16_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 db;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kUmmaDescHigh)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(smem_dst), "l"(map), "r"(bar), "r"(x),
               "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two floats in one operation (the same roundings as one at a time).
struct Pair {
  unsigned long long bits;
};
__device__ __forceinline__ Pair pair_of(float low, float high) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r.bits) : "f"(low), "f"(high));
  return r;
}
__device__ __forceinline__ void unpair(Pair v, float& low, float& high) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(low), "=f"(high) : "l"(v.bits)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}

// A whole warp waits: what follows is warp-wide, so the lanes go on or give up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
}

struct PrefixTCParams {
  int num_pages;
  const int* positions;
  const int* seq_starts;
  const int* block_table;
  int table_stride;
  __nv_bfloat16* out;     // OWN: finished rows [rows, q heads * head size]
  float* part_o;          // [rows, q heads, parts, head size]: written, or with OWN read (parts 0: none)
  float2* part_ml;        // [rows, q heads, parts]
  int parts, rows, entries, q_heads, kv_heads, page_size, box_keys, shared, first_key;
  float scale;
  int* error_flag;
};

template <int D>
struct SmemPrefix {
  static constexpr int kStages = D <= 64 ? 3 : 2;
  // 1024-byte aligned, each a run of sub-tiles [rows][64] of 64 dims in the 128-byte swizzle
  __nv_bfloat16 q[2][kPairsTC * D];
  __nv_bfloat16 k[kStages][kKeysTC * D];
  __nv_bfloat16 v[kStages][kKeysTC * D];
  int bad[3][D];                 // per dim the first key whose value is +infinity, -infinity, NaN and was taken out
  int lowest[2], last[2];        // the fewest and the most keys that a row of each row tile sees
  int entry, token0, tokens;     // OWN: whose rows, the first one of this CTA, how many
  int any_bad;
  // k_full, v_full: a tile has landed.  k_empty, v_empty: both row tiles' products have read it.  s_full: a row tile's scores are there.  p_full: a half of its weights is.  pv_done:
  // its weighted values are added.
  uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_full[2][2], pv_done[2];
  uint32_t tmem_base;
  int abort_flag;
};

template <int D, bool OWN>
__global__ void __launch_bounds__(kThreadsTC, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, const PrefixTCParams p) {
  extern __shared__ uint8_t smem_raw[];
  using Smem = SmemPrefix<D>;
  constexpr int kStages = Smem::kStages, kHalves = D / kBoxDims;
  Smem& sm = *reinterpret_cast<Smem*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = OWN ? blockIdx.x : blockIdx.y;
  const int group = p.q_heads / p.kv_heads, tile_tokens = kPairsTC / group;
  constexpr int kTmemCols = 512, kOutCol0 = 256;   // S of the two row tiles at 0 and 128, their outputs at 256 and 384

  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.k_empty[s], 2);
      mbar_init(&sm.v_empty[s], 2);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&sm.s_full[u], 1);
      mbar_init(&sm.pv_done[u], 1);
      mbar_init(&sm.p_full[u][0], 4);   // one arrival per softmax warp
      mbar_init(&sm.p_full[u][1], 4);
      sm.lowest[u] = kNoKey;
      sm.last[u] = 0;
    }
    sm.abort_flag = sm.any_bad = 0;
    sm.entry = sm.token0 = sm.tokens = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  for (int i = threadIdx.x; i < 3 * D; i += kThreadsTC) (&sm.bad[0][0])[i] = kNoKey;
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sm.tmem_base)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem = sm.tmem_base;
  // Nothing of global memory is touched before the kernel in front has completed.  With OWN and parts that one is the prefix's, which lets this one start when all
  // its CTAs are past this very wait: then what came before it is complete, and only its parts have to be waited for, at the end.
  const bool waits_late = OWN && p.parts > 0;
  if (!waits_late) grid_dependency_wait();
  if (!OWN) grid_launch_dependents();

  // which rows: token0, and up to 2 * tile_tokens rows from there
  const int first_row = max(0, p.seq_starts[0]), end_row = min(p.rows, p.seq_starts[p.entries]);
  int token0, tokens, entry = 0;
  if (OWN) {
    if (warp == 0) {   // the entry that this CTA's number falls to, counting every entry's pairs of row tiles: 32 entries at a time
      const int wanted = blockIdx.y, each = 2 * tile_tokens;
      int before = 0;
      for (int e0 = 0; e0 < p.entries; e0 += 32) {
        const int e = e0 + lane;
        int begin = 0, end = 0;
        if (e < p.entries) {
          begin = max(first_row, p.seq_starts[e]);
          end = min(end_row, p.seq_starts[e + 1]);
        }
        const int pieces = end > begin ? (end - begin + each - 1) / each : 0;
        int upto = pieces;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, upto, offset);
          if (lane >= offset) upto += other;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > wanted);
        if (past != 0u) {
          if (lane == __ffs(past) - 1) {
            sm.entry = e;
            sm.token0 = begin + (wanted - (before + upto - pieces)) * each;
            sm.tokens = min(each, end - sm.token0);
          }
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    __syncthreads();
    entry = sm.entry, token0 = sm.token0, tokens = sm.tokens;
  } else {
    token0 = first_row + (int)blockIdx.z * 2 * tile_tokens;
    tokens = max(0, min(2 * tile_tokens, end_row - token0));
  }
  const int* table = p.block_table + (size_t)entry * p.table_stride;
  const long long room = (long long)p.table_stride * p.page_size;
  // keys that a row of the step sees in this kind of part: those below the result
  auto limit_of = [&](int token) {
    long long seen = (long long)p.positions[token] + 1;
    if (seen > room) {
      atomicOr(p.error_flag, kBadPage);
      seen = room;
    }
    return (int)max(0ll, OWN ? seen : min(seen, (long long)p.shared));
  };
  for (int i = threadIdx.x; i < tokens; i += kThreadsTC) {
    const int limit = limit_of(token0 + i), u = i >= tile_tokens;
    atomicMin(&sm.lowest[u], limit);
    atomicMax(&sm.last[u], limit);
  }
  __syncthreads();
  // key tiles: of the prefix a run of them per CTA
  const int last = max(sm.last[0], sm.last[1]);
  int kt_begin = OWN ? p.first_key / kKeysTC : 0, kt_end = (last + kKeysTC - 1) / kKeysTC;
  if (!OWN) {
    const int all = (p.shared + kKeysTC - 1) / kKeysTC;
    kt_begin = (int)((long long)all * blockIdx.x / gridDim.x);
    kt_end = min(kt_end, (int)((long long)all * (blockIdx.x + 1) / gridDim.x));
  }
  auto tiles_of = [&](int u) { return max(0, min(kt_end, (sm.last[u] + kKeysTC - 1) / kKeysTC) - kt_begin); };
  const int n0 = tiles_of(0), n1 = tiles_of(1), n = max(n0, n1);

  if (warp < kFirstSoftmaxWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kControlRegs));
  if (warp == 0) {
    if (n > 0 && lane == 0) {   // Q: per row tile and 64 dims one box of the group's heads of tile_tokens rows
      const uint32_t bytes = (uint32_t)tile_tokens * group * kBoxDims * 2 * kHalves;
      const int row_tiles = tokens > tile_tokens ? 2 : 1;
      mbar_expect_tx(smem_u32(&sm.q_full), bytes * row_tiles);
      for (int u = 0; u < row_tiles; ++u)
#pragma unroll
        for (int c = 0; c < kHalves; ++c)
          tma_load_3d(smem_u32(sm.q[u]) + c * (kPairsTC * kBoxDims * 2), &map_q, c * kBoxDims, kvh * group, token0 + u * tile_tokens, smem_u32(&sm.q_full));
    }
    // A key tile is `boxes` boxes of box_keys keys in each half of the dims; lane i copies box i % boxes of half i / boxes.
    const int boxes = kKeysTC / p.box_keys, box = lane % boxes, half = lane / boxes;
    const bool copies = half < kHalves;
    const int rows_of_pool = p.num_pages * 2 * p.kv_heads * p.page_size;   // (the host has seen that this fits)
    RingPosition<kStages> ring;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j, ring.advance()) {
      const int key = (kt_begin + j) * kKeysTC + box * p.box_keys;
      int row = rows_of_pool, value_row = rows_of_pool;   // past the last key nothing is read: zeros arrive
      if (copies && key < last) {
        int page = table[key / p.page_size];
        if ((unsigned)page >= (unsigned)p.num_pages) {   // reported, and page 0 read in its place
          atomicOr(p.error_flag, kBadPage);
          page = 0;
        }
        row = (page * 2 * p.kv_heads + kvh) * p.page_size + key % p.page_size;
        value_row = row + p.kv_heads * p.page_size;
      }
      const uint32_t offset = ring.stage * (kKeysTC * D * 2) + half * (kKeysTC * kBoxDims * 2) + box * p.box_keys * (kBoxDims * 2);
      ok = warp_wait(&sm.k_empty[ring.stage], ring.phase ^ 1, abort_flag);
      if (lane == 0 && ok) mbar_expect_tx(&sm.k_full[ring.stage], kKeysTC * D * 2);
      __syncwarp();
      if (ok && copies) tma_load_2d(smem_u32(sm.k) + offset, &map_kv, half * kBoxDims, row, smem_u32(&sm.k_full[ring.stage]));
      if (ok) ok = warp_wait(&sm.v_empty[ring.stage], ring.phase ^ 1, abort_flag);
      if (lane == 0 && ok) mbar_expect_tx(&sm.v_full[ring.stage], kKeysTC * D * 2);
      __syncwarp();
      if (ok && copies) tma_load_2d(smem_u32(sm.v) + offset, &map_kv, half * kBoxDims, value_row, smem_u32(&sm.v_full[ring.stage]));
    }
  } else if (warp < 3) {
    if (lane == 0) {   // the products of row tile u
      const int u = warp - 1, mine = u == 0 ? n0 : n1;
      constexpr uint32_t idesc_s = umma_instr_desc(kPairsTC, kKeysTC), idesc_pv = instr_desc_b_mn(kPairsTC, D);
      constexpr uint32_t kSub = (kKeysTC * kBoxDims * 2) >> 4;   // one sub-tile of 64 dims further, in descriptor units (Q's and K's alike)
      // V is the MN-major operand: beyond 64 dims the next sub-tile lies kSub on, which the leading-dimension offset says; one sub-tile needs none
      constexpr uint32_t kVLeading = kHalves > 1 ? kSub : 1u;
      const uint32_t q_low = umma_desc_low(smem_u32(sm.q[u])), k_low = umma_desc_low(smem_u32(sm.k));
      const uint32_t v_low = ((smem_u32(sm.v) >> 4) & 0x3FFF) | (kVLeading << 16);
      const uint32_t tmem_s = tmem + u * kKeysTC, tmem_o = tmem + kOutCol0 + u * 128;
      RingPosition<kStages> ring;
      bool ok = mine == 0 || mbar_wait(&sm.q_full, 0, abort_flag);
      for (int j = 0; j < n && ok; ++j, ring.advance()) {
        ok = mbar_wait(&sm.k_full[ring.stage], ring.phase, abort_flag);
        if (ok && j >= mine) {   // none of this tile's rows sees these keys
          mbar_arrive(&sm.k_empty[ring.stage]);
          ok = mbar_wait(&sm.v_full[ring.stage], ring.phase, abort_flag);
          if (ok) mbar_arrive(&sm.v_empty[ring.stage]);
          continue;
        }
        if (ok && j > 0) ok = mbar_wait(&sm.pv_done[u], (j - 1) & 1, abort_flag);   // the weights that lie over the scores have been read
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const uint32_t k_tile = k_low + ring.stage * ((kKeysTC * D * 2) >> 4), v_tile = v_low + ring.stage * ((kKeysTC * D * 2) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)   // 16 dims further: 32 bytes inside a sub-tile's rows, then the next sub-tile
          umma_bf16(tmem_s, q_low + (kk >> 2) * kSub + (kk & 3) * 2, k_tile + (kk >> 2) * kSub + (kk & 3) * 2, idesc_s, kk > 0 ? 1u : 0u);
        umma_commit(&sm.s_full[u]);
        umma_commit(&sm.k_empty[ring.stage]);
        ok = mbar_wait(&sm.v_full[ring.stage], ring.phase, abort_flag);
#pragma unroll
        for (int h = 0; h < 2 && ok; ++h) {
          ok = mbar_wait(&sm.p_full[u][h], j & 1, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
          for (int kk = 4 * h; kk < 4 * h + 4; ++kk)   // 16 keys further: 8 columns of P, 16 rows (2048 bytes) down in a V sub-tile
            umma_bf16_a_tmem(tmem_o, tmem_s + kk * 8, v_tile + kk * ((16 * kBoxDims * 2) >> 4), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
        }
        if (!ok) break;
        umma_commit(&sm.v_empty[ring.stage]);
        umma_commit(&sm.pv_done[u]);
      }
    }
  } else if (warp >= kFirstSoftmaxWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
    const int u = (warp - kFirstSoftmaxWarp) >> 2, sub = warp & 3, pair = sub * 32 + lane, mine = u == 0 ? n0 : n1;
    const uint32_t lane_base = (uint32_t)(sub * 32) << 16;
    const uint32_t tmem_s = tmem + lane_base + u * kKeysTC, tmem_o = tmem + lane_base + kOutCol0 + u * 128;
    const int tile_rows = max(0, min(tile_tokens, tokens - u * tile_tokens));
    const bool mine_valid = pair < tile_rows * group;
    const int token = token0 + u * tile_tokens + pair / group, head = kvh * group + pair % group;
    const int limit = mine_valid ? limit_of(token) : 0;
    const int lowest = sm.lowest[u];
    const float sl2 = p.scale * kToLog2;
    float reference = -INFINITY, row_sum = 0.0f;
    RingPosition<kStages> at;
    bool ok = true;
    for (int j = 0; j < mine && ok; ++j, at.advance()) {
      const int key0 = (kt_begin + j) * kKeysTC;
      ok = warp_wait(&sm.s_full[u], j & 1, abort_flag);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      float sc[kKeysTC];
      tmem_ld64(tmem_s, sc);
      tmem_ld64(tmem_s + 64, sc + 64);
      const bool masked = key0 + kKeysTC > lowest || (OWN && key0 < p.first_key);
      if (masked) {
#pragma unroll
        for (int i = 0; i < kKeysTC; ++i) sc[i] = key0 + i < limit && (!OWN || key0 + i >= p.first_key) ? sc[i] : -INFINITY;
      }
      float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
      for (int i = 0; i < kKeysTC; i += 8) {
        m0 = max3(m0, sc[i], sc[i + 1]);
        m1 = max3(m1, sc[i + 2], sc[i + 3]);
        m2 = max3(m2, sc[i + 4], sc[i + 5]);
        m3 = max3(m3, sc[i + 6], sc[i + 7]);
      }
      const float scaled_max = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * sl2;
      if (j == 0) {
        reference = scaled_max;
      } else {
        // The output and the sum are taken against `reference`.  (The product that last added to the output is done: the scores waited for were issued behind it.)
        const bool grown = scaled_max > reference + kLazyRescale;
        if (__any_sync(0xffffffffu, grown)) {
          const float alpha = grown ? exp2f(reference - scaled_max) : 1.0f;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_load_32(tmem_o + c * 32, o);
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_store_32(tmem_o + c * 32, o);
          }
          row_sum *= alpha;
          if (grown) reference = scaled_max;
        }
      }
      const float base = reference == -INFINITY ? 0.0f : reference;   // a row that has seen no key yet: every weight is 0
      if (masked) {
        // Values of keys that none of the CTA's rows sees (never written, perhaps) become zeros: 0 * (whatever is there) must stay 0.  Of keys that some rows see, what is
        // not finite is taken out and noted.
        const bool some_see = lowest < min(key0 + kKeysTC, last);
        const int none_from = max(0, min(kKeysTC, last - key0)), none_to = OWN ? max(0, min(kKeysTC, p.first_key - key0)) : 0;
        if (none_from < kKeysTC || none_to > 0 || some_see) {
          ok = warp_wait(&sm.v_full[at.stage], at.phase, abort_flag);
          if (!ok) break;
          uint8_t* v_tile = reinterpret_cast<uint8_t*>(sm.v[at.stage]);
          for (int r = pair >> 3; r < kKeysTC; r += kPairsTC / 8) {   // 8 threads a row of 128 bytes, whatever the swizzle
            if (r < none_to || r >= none_from) {
#pragma unroll
              for (int c = 0; c < kHalves; ++c) *reinterpret_cast<uint4*>(v_tile + c * (kKeysTC * kBoxDims * 2) + r * 128 + (pair & 7) * 16) = make_uint4(0, 0, 0, 0);
            } else if (some_see) {
#pragma unroll
              for (int c = 0; c < kHalves; ++c) {
                uint16_t* chunk = reinterpret_cast<uint16_t*>(v_tile + c * (kKeysTC * kBoxDims * 2) + r * 128 + (pair & 7) * 16);
                const uint4 eight = *reinterpret_cast<const uint4*>(chunk);
                const uint32_t words[4] = {eight.x, eight.y, eight.z, eight.w};
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                  const uint32_t bits = (words[w >> 1] >> (16 * (w & 1))) & 0xffffu;
                  if ((bits & 0x7f80u) == 0x7f80u) {
                    const int dim = c * kBoxDims + (((pair & 7) ^ (r & 7)) << 3) + w;   // the 128-byte swizzle: chunk i of row r lies at i ^ (r % 8)
                    atomicMin(&sm.bad[(bits & 0x7fu) != 0u ? 2 : (bits >> 15)][dim], key0 + r);
                    sm.any_bad = 1;
                    __threadfence_block();
                    chunk[w] = 0;
                  }
                }
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // generic-proxy writes -> visible to the tensor core
        }
      }
      const Pair scale2 = pair_of(sl2, sl2), minus_base2 = pair_of(-base, -base);
      Pair sums = pair_of(0.0f, 0.0f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t packed[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float x0, x1;
          unpair(fma2(pair_of(sc[64 * h + 2 * i], sc[64 * h + 2 * i + 1]), scale2, minus_base2), x0, x1);
          const float p0 = exp2_approx(x0), p1 = exp2_approx(x1);
          sums = add2(sums, pair_of(p0, p1));
          packed[i] = pack_bf16(p0, p1);   // a weight keeps 8 bits where it meets its value, as in the other bfloat16 attention kernels; the sum has all of it
        }
        tmem_store_32(tmem_s + 32 * h, packed);   // over scores that are in registers by now
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[u][h]);
      }
      float sum0, sum1;
      unpair(sums, sum0, sum1);
      row_sum += sum0 + sum1;
    }
    if (ok && mine > 0) ok = warp_wait(&sm.pv_done[u], (mine - 1) & 1, abort_flag);
    if (waits_late) grid_dependency_wait();   // the prefix's parts
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const size_t at_pair = (size_t)token * p.q_heads + head;
      const bool any_bad = *(volatile int*)&sm.any_bad != 0;
      float top = reference, total = row_sum, factor = 1.0f;
      if (OWN && mine_valid) {
        for (int i = 0; i < p.parts; ++i) top = fmaxf(top, __ldcg(&p.part_ml[at_pair * p.parts + i]).x);
        factor = reference == -INFINITY ? (row_sum == 0.0f ? 0.0f : 1.0f) : exp2f(reference - top);   // (a part of nothing but NaN keeps its NaN)
        total = row_sum * factor;
        for (int i = 0; i < p.parts; ++i) {
          const float2 ml = __ldcg(&p.part_ml[at_pair * p.parts + i]);
          const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2f(ml.x - top);
          if (f != 0.0f) total = fmaf(f, ml.y, total);
        }
      } else if (mine_valid) {
        p.part_ml[at_pair * p.parts + blockIdx.x] = make_float2(reference, row_sum);
      }
      const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {   // 32 columns at a time (the load is warp-wide: every lane takes part)
        uint32_t raw[32];
        if (mine > 0) {
          tmem_load_32(tmem_o + c * 32, raw);
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
        }
        if (!mine_valid) continue;
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = mine > 0 ? __uint_as_float(raw[i]) : 0.0f;
        if (any_bad) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const volatile int* first = &sm.bad[0][c * 32 + i];
            const bool plus = first[0] < limit, minus = first[D] < limit, none = first[2 * D] < limit;
            if (none || (plus && minus)) o[i] = __int_as_float(0x7fffffff);
            else if (plus) o[i] += INFINITY;
            else if (minus) o[i] -= INFINITY;
          }
        }
        if (OWN) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = factor == 0.0f ? 0.0f : o[i] * factor;
          for (int s = 0; s < p.parts; ++s) {
            const float2 ml = __ldcg(&p.part_ml[at_pair * p.parts + s]);
            const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2f(ml.x - top);
            if (f == 0.0f) continue;
            const float4* part = reinterpret_cast<const float4*>(p.part_o + (at_pair * p.parts + s) * D + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 v = __ldcg(part + i);
              o[4 * i] = fmaf(f, v.x, o[4 * i]), o[4 * i + 1] = fmaf(f, v.y, o[4 * i + 1]), o[4 * i + 2] = fmaf(f, v.z, o[4 * i + 2]), o[4 * i + 3] = fmaf(f, v.w, o[4 * i + 3]);
            }
          }
          uint4* to = reinterpret_cast<uint4*>(p.out + at_pair * D + c * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            to[i] = make_uint4(pack_bf16(o[8 * i] * inverse, o[8 * i + 1] * inverse), pack_bf16(o[8 * i + 2] * inverse, o[8 * i + 3] * inverse),
                               pack_bf16(o[8 * i + 4] * inverse, o[8 * i + 5] * inverse), pack_bf16(o[8 * i + 6] * inverse, o[8 * i + 7] * inverse));
        } else if (mine > 0) {
          float4* to = reinterpret_cast<float4*>(p.part_o + (at_pair * p.parts + blockIdx.x) * D + c * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  }
  close_and_report(abort_flag, p.error_flag);
  if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols));
}

// q heads of rows q_row_stride elements apart as [rows][heads][dim], a box the group's heads of `tile_tokens` rows.
static bool make_q_map(CUtensorMap* map, const void* q, int rows, int q_heads, int dim, long long q_row_stride, int group, int tile_tokens) {
  EncodeTiledFn fn = encode_tiled();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)q_heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)q_row_stride * 2};
  const cuuint32_t box[3] = {(cuuint32_t)kBoxDims, (cuuint32_t)group, (cuuint32_t)tile_tokens};
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool OWN>
static int launch_tc(const CUtensorMap& map_q, const CUtensorMap& map_kv, const PrefixTCParams& p, dim3 grid, cudaStream_t stream) {
  static std::atomic<unsigned long long> devices{0};
  static std::atomic<int> registers{0};
  const int smem = (int)sizeof(SmemPrefix<D>) + 1024;
  cudaError_t e = allow_shared_memory(prefix_tc_kernel<D, OWN>, smem, devices);
  if (e != cudaSuccess) return (int)e;
  if (registers.load(std::memory_order_relaxed) == 0) {   // the warps' shares are handed out of what the launch holds: less than that would wait for good
    cudaFuncAttributes found;
    e = cudaFuncGetAttributes(&found, prefix_tc_kernel<D, OWN>);
    if (e != cudaSuccess) return (int)e;
    registers.store(found.numRegs, std::memory_order_relaxed);
  }
  if (registers.load(std::memory_order_relaxed) < kLaunchRegs) return (int)cudaErrorLaunchOutOfResources;
  return (int)launch_pdl(prefix_tc_kernel<D, OWN>, grid, dim3(kThreadsTC), (size_t)smem, stream, map_q, map_kv, p);
}

}  // namespace tlie

using namespace tlie;

// q: rows [rows, q_row_stride] that start with the (rotated) query heads.  pages: one layer's pool [num_pages, 2, kv_heads, page_size, head_dim].
// own 0: the parts of the keys below `shared`, cut into `parts` runs, into part_ml [rows, q_heads, parts, 2] and part_o [rows, q_heads, parts, head_dim] (a part without keys
// leaves part_o as it is).  own 1: out [rows, q_heads * head_dim] from the keys from first_key on and, if parts > 0, the parts of those below, which the kernel
// in front in the stream must write.  Rows outside [seq_starts[0], seq_starts[entries]) are left as they are.
TLIE_EXPORT int tlie_prefix_tc(int own, const void* q, long long q_row_stride, const void* pages, int num_pages, const int* positions, const int* seq_starts,
                               const int* block_table, int table_stride, void* out, float* part_ml, float* part_o, int parts, int rows, int entries, int q_heads, int kv_heads,
                               int head_dim, int page_size, int shared, int first_key, float scale, int* error_flag, cudaStream_t stream) {
  if (rows <= 0 || entries <= 0) return 0;
  if (kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > kPairsTC || kv_heads > 65535 || page_size <= 0 || page_size % 16 != 0 || num_pages <= 0 || q_row_stride % 8 != 0 ||
      (head_dim != 64 && head_dim != 128) || error_flag == nullptr || ((uintptr_t)q & 15) || ((uintptr_t)pages & 15) || ((uintptr_t)out & 15) || ((uintptr_t)part_o & 15) ||
      ((uintptr_t)part_ml & 7) || (!own && (parts < 1 || shared < 1)))
    return (int)cudaErrorInvalidValue;
  const int group = q_heads / kv_heads, tile_tokens = kPairsTC / group;
  const long long pool_rows = (long long)num_pages * 2 * kv_heads * page_size;
  if (pool_rows >= 0x7fffffffLL - 256) return (int)cudaErrorInvalidValue;   // a copy's row is a 32-bit coordinate
  int box_keys = 16;
  while (box_keys < kKeysTC && page_size % (2 * box_keys) == 0) box_keys *= 2;
  CUtensorMap map_q, map_kv;
  if (!make_q_map(&map_q, q, rows, q_heads, head_dim, q_row_stride, group, tile_tokens) || !make_map(&map_kv, pages, (int)pool_rows, head_dim, box_keys))
    return (int)cudaErrorInvalidValue;
  PrefixTCParams p{num_pages, positions, seq_starts, block_table, table_stride, (__nv_bfloat16*)out, part_o, (float2*)part_ml, parts, rows, entries, q_heads, kv_heads, page_size,
                   box_keys, shared, first_key, scale, error_flag};
  const int pieces = (rows + 2 * tile_tokens - 1) / (2 * tile_tokens);
  if (own) {
    const long long items = (long long)rows / (2 * tile_tokens) + entries;   // every entry may leave one piece that is not full
    if (items > 65535) return (int)cudaErrorInvalidValue;
    const dim3 grid(kv_heads, (unsigned)items);
    return head_dim == 64 ? launch_tc<64, true>(map_q, map_kv, p, grid, stream) : launch_tc<128, true>(map_q, map_kv, p, grid, stream);
  }
  if (pieces > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid(parts, kv_heads, pieces);
  return head_dim == 64 ? launch_tc<64, false>(map_q, map_kv, p, grid, stream) : launch_tc<128, false>(map_q, map_kv, p, grid, stream);
}
