// Paged grouped-query attention for batches whose requests share their first cached keys, on the 5th-generation tensor cores (bfloat16, head size 64 or 128,
// pages of a multiple of 16 keys).  Three builds of one kernel:
//   * of the prefix: all rows of the step against the keys below `shared`, a run of which a CTA takes; it leaves (m, l, o) per (row, query head): the
//     largest score (a reference near it), the sum of weights and the weighted sum of values;
//   * of an entry's own keys (OWN): an entry's rows against its keys first_key <= j <= p, to the finished output, brought together with the parts of the prefix
//     (JOINS); without them first_key is 0, and this is the whole attention of portions of many rows.
//
// The query heads of a group meet the same keys: a row tile is 128 (row, head of the group) pairs, 128 / group rows of the step.  A CTA has two such tiles and a
// ring of key and value tiles for both, so that keys and values come from L2 once per 256 pairs.  One CTA fills an SM.
//   * TMA brings Q once (a box of 64 dims x the group's heads x 128 / group rows per half), and every key tile as boxes that lie inside a page.  The lanes of
//     the producing warp each look up one box's page and copy it;
//   * S = Q . K^T (a warp per row tile) and O += P . V are issued by warps of their own.  P has a place of its own in tensor memory: scores may be written again as soon as the softmax threads
//     have them in registers, so the next scores are computed under this tile's softmax, and a softmax thread finds its next scores waiting.  With the weights over
//     the scores (128 keys at both head sizes), scores, softmax and weighted values of a row tile were a chain that the other tile's could only half
//     fill: 3,900 cycles per 128 keys and two row tiles at head size 128, where the tensor core has 2,050 and the exponential unit 2,050 to do.  512 columns of tensor
//     memory hold, twice, output, scores and weights of 64 dims and 128 keys, or of 128 dims and 80 keys;
//   * thread = (row, head) pair = lane of tensor memory: maxima and sums need no other thread.  The output is taken against a reference maximum that
//     moves only when a tile's maximum is more than 2^8 above it;
//   * what a tile's rows do not all see is masked; a value that some of them see and that is not finite would spread through a weight of zero, so in such tiles values are looked
//     through, what is not finite is taken out and noted, and the rows that do see it show it in the end.
// A key tile of two row tiles takes 1.05 us at head size 128 (80 keys) and 1.7 at 64 (128 keys): 148 SMs then do 1,480 TFLOP/s, 0.93 of the measured rate of large products.  An item costs 4 us more,
// and 4 pass before the first.  Portions (1,781 rows of 8 entries, 8 key/value heads of 128 for 4 query heads each, 4,096 shared keys and up to 256 own) take 139 us for 122.8 GFLOP (884 TFLOP/s: items of
// part of 256 pairs, and 1.9 rounds of them).  256 rows against 24,576 shared keys: 97 us for 103 GFLOP on 128 of 148 SMs.
// Every wait is bounded; a CTA that gives up raises the device's error word, lets its copies land and returns.
#include <type_traits>

#include "shared_memory_limit.cuh"
#include "tcgen05_utils.cuh"

namespace tlie {

constexpr int kPairsTC = 128;       // (row, head) pairs of a row tile
constexpr int kBoxDims = 64;        // dims of one box: 128 bytes, the swizzle span
constexpr int kThreadsTC = 512;     // warps 0 copies keys, 1 values, 2 and 3 scores of the two row tiles, 4 weighted values, 5 to 7 none, 8 to 11 and 12 to 15 softmax of the row tiles
constexpr int kFirstSoftmaxWarp = 8;
constexpr int kControlRegs = 56, kSoftmaxRegs = 200, kLaunchRegs = 128;   // 256 * 56 + 256 * 200 = 512 * 128
constexpr float kToLog2 = 1.4426950408889634f;
constexpr float kLazyRescale = 8.0f;
constexpr int kBadPage = 8;         // the bit of the device's error word
constexpr int kNoKey = 0x7fffffff;

// bf16 x bf16 -> f32, A K-major, B MN-major (V stays [key][dim], as the cache stores it), tile m x n.
__host__ __device__ constexpr uint32_t instr_desc_b_mn(int m, int n) { return umma_instr_desc(m, n) | (1u << 16); }

// Columns of this thread's lane written from registers (not waited for).
__device__ __forceinline__ void tmem_store_8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_store_4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// ... and read into them (not waited for).
__device__ __forceinline__ void tmem_load_8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// The four softmax warps of row tile u meet.
__device__ __forceinline__ void tile_barrier(int u) { asm volatile("bar.sync %0, 128;\n" ::"r"(1 + u) : "memory"); }
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

// One lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(elected));
  return elected != 0;
}

// A whole warp waits: what follows is warp-wide, so the lanes go on or give up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(bar, parity)), 1)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, gave_up)) != 0;
}

// Non-zero where one of two bfloat16 numbers is infinite or NaN (an exponent of ones carries into the sign's place).
__device__ __forceinline__ uint32_t not_finite(uint32_t two) { return ((two & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
// Of eight values of a key those that are not finite become zero, and the first such key is noted per dim: at bad[dim] for +infinity, `dims` further for -infinity, as much
// again for NaN.
__device__ __forceinline__ void take_out(uint16_t* eight, int* bad, int dims, int key, int* any_bad) {
#pragma unroll 1
  for (int w = 0; w < 8; ++w) {
    const uint32_t bits = eight[w];
    if ((bits & 0x7f80u) != 0x7f80u) continue;
    atomicMin(bad + ((bits & 0x7fu) != 0u ? 2 : bits >> 15) * dims + w, key);
    *(volatile int*)any_bad = 1;
    __threadfence_block();
    eight[w] = 0;
  }
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
constexpr int kKeysOf = D <= 64 ? 128 : 80;   // keys of a key tile

// Parts of the prefix that a CTA of own keys brings together: their factors lie in Q's place, behind 16 columns of a row tile's output.
template <int D>
constexpr int kOwnParts = (D * 2 - 64) / 4 < 32 ? (D * 2 - 64) / 4 : 32;

template <int D>
struct SmemPrefix {
  static constexpr int kKeys = kKeysOf<D>, kStages = D <= 64 ? 4 : 3;
  // 1024-byte aligned, each a run of sub-tiles [rows][64] of 64 dims in the 128-byte swizzle
  __nv_bfloat16 q[2][kPairsTC * D];
  __nv_bfloat16 k[kStages][kKeys * D];
  __nv_bfloat16 v[kStages][kKeys * D];
  int bad[3][D];                 // per dim the first key whose value is +infinity, -infinity, NaN and was taken out
  int lowest[2], last[2];        // the fewest and the most keys that a row of each row tile sees
  int entry, token0, tokens;     // OWN: whose rows, the first one of this CTA, how many
  int any_bad;
  // k_full, v_full: a tile has landed.  k_empty, v_empty: both row tiles' products have read it.  s_full: a row tile's scores are there; s_read: its threads have
  // them.  p_full: its weights are there; pv_done: its weighted values are added.
  uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], s_read[2], p_full[2], pv_done[2], exps_done[2][4];
  uint32_t tmem_base;
  int gave_up;
};

template <int D, bool OWN, bool JOINS>
__global__ void __launch_bounds__(kThreadsTC, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, const PrefixTCParams p) {
  extern __shared__ uint8_t smem_raw[];
  using Smem = SmemPrefix<D>;
  constexpr int kStages = Smem::kStages, kKeys = Smem::kKeys, kHalves = D / kBoxDims;
  Smem& sm = *reinterpret_cast<Smem*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  volatile int* gave_up = &sm.gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = OWN ? blockIdx.x : blockIdx.y;
  const int group = p.q_heads / p.kv_heads, tile_tokens = kPairsTC / group;
  // tensor memory: the two row tiles' outputs, scores and weights (two keys a column)
  constexpr int kTmemCols = 512, kScoreCol0 = 2 * D, kWeightCol0 = kScoreCol0 + 2 * kKeys, kWeightCols = (kKeys / 2 + 15) / 16 * 16;
  static_assert(kWeightCol0 + 2 * kWeightCols <= kTmemCols && kKeys % 16 == 0, "tensor memory holds 512 columns");

  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.k_empty[s], 2);   // a commit per row tile
      mbar_init(&sm.v_empty[s], 1);
    }
    for (int u = 0; u < 2; ++u) {
      for (int w = 0; w < 4; ++w) mbar_init(&sm.exps_done[u][w], 1);
      mbar_init(&sm.s_full[u], 1);
      mbar_init(&sm.pv_done[u], 1);
      mbar_init(&sm.s_read[u], 4);   // one arrival per softmax warp
      mbar_init(&sm.p_full[u], 4);
      sm.lowest[u] = kNoKey;
      sm.last[u] = 0;
    }
    sm.gave_up = sm.any_bad = 0;
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
  // Nothing of global memory is touched before the kernel in front has completed.  With JOINS that one is the prefix's, which lets this one start when all
  // its CTAs are past this very wait: then what came before it is complete, and only its parts have to be waited for, at the end.
  if (!JOINS) grid_dependency_wait();
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
  // Key tiles.  Of the prefix a run of them per CTA, whichever rows see them: nothing has to wait for the rows' positions then.  Of an entry's own keys those that some row sees.
  int kt_begin, n0, n1, last;
  if (OWN) {
    for (int i = threadIdx.x; i < tokens; i += kThreadsTC) {
      const int limit = limit_of(token0 + i), u = i >= tile_tokens;
      atomicMin(&sm.lowest[u], limit);
      atomicMax(&sm.last[u], limit);
    }
    __syncthreads();
    last = max(sm.last[0], sm.last[1]);
    kt_begin = p.first_key / kKeys;
    n0 = max(0, (sm.last[0] + kKeys - 1) / kKeys - kt_begin);
    n1 = max(0, (sm.last[1] + kKeys - 1) / kKeys - kt_begin);
  } else {
    const int all = (p.shared + kKeys - 1) / kKeys;
    last = p.shared;
    kt_begin = (int)((long long)all * blockIdx.x / gridDim.x);
    const int mine = (int)((long long)all * (blockIdx.x + 1) / gridDim.x) - kt_begin;
    n0 = tokens > 0 ? mine : 0;
    n1 = tokens > tile_tokens ? mine : 0;
  }
  const int n = max(n0, n1);

  if (warp < kFirstSoftmaxWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kControlRegs));
  if (warp < 2) {
    if (warp == 0 && n > 0 && lane == 0) {   // Q: per row tile and 64 dims one box of the group's heads of tile_tokens rows
      const uint32_t bytes = (uint32_t)tile_tokens * group * kBoxDims * 2 * kHalves;
      const int row_tiles = tokens > tile_tokens ? 2 : 1;
      mbar_expect_tx(smem_u32(&sm.q_full), bytes * row_tiles);
      for (int u = 0; u < row_tiles; ++u)
#pragma unroll
        for (int c = 0; c < kHalves; ++c)
          tma_load_3d(smem_u32(sm.q[u]) + c * (kPairsTC * kBoxDims * 2), &map_q, c * kBoxDims, kvh * group, token0 + u * tile_tokens, smem_u32(&sm.q_full));
    }
    // A warp for keys and one for values: a copy costs the warp that issues it some 85 cycles, and a tile of 80 keys is five boxes in each half of the dims.  Lane i looks up where
    // box i lies in the pool, a tile ahead; one lane copies them all.
    constexpr int kMostBoxes = kKeys % 128 == 0 ? 8 : kKeys / 16;
    const int boxes = kKeys / p.box_keys, box_bytes = p.box_keys * kBoxDims * 2, further = warp * p.kv_heads * p.page_size;   // values lie behind a page's keys
    const int rows_of_pool = p.num_pages * 2 * p.kv_heads * p.page_size;   // (the host has seen that this fits)
    const uint32_t tiles = smem_u32(warp == 0 ? sm.k[0] : sm.v[0]);
    uint64_t* const full = warp == 0 ? sm.k_full : sm.v_full;
    uint64_t* const empty = warp == 0 ? sm.k_empty : sm.v_empty;
    const bool leader = elect_one();
    auto look_up = [&](int j) {
      const int key = (kt_begin + j) * kKeys + lane * p.box_keys;
      if (lane >= boxes || key >= last) return rows_of_pool;   // past the last key nothing is read: zeros arrive
      const int index = key / p.page_size;
      int page = table[index];
      if ((unsigned)page >= (unsigned)p.num_pages) {   // reported, and page 0 read in its place
        atomicOr(p.error_flag, kBadPage);
        page = 0;
      }
      return (page * 2 * p.kv_heads + kvh) * p.page_size + (key - index * p.page_size) + further;
    };
    RingPosition<kStages> ring;
    bool ok = true;
    int rows = n > 0 ? look_up(0) : 0;
    for (int j = 0; j < n && ok; ++j, ring.advance()) {
      ok = warp_wait(&empty[ring.stage], ring.phase ^ 1, gave_up);
      if (!ok) break;
      const uint32_t to = tiles + ring.stage * (kKeys * D * 2), bar = smem_u32(&full[ring.stage]);
      if (leader) mbar_expect_tx(bar, kKeys * D * 2);
#pragma unroll
      for (int b = 0; b < kMostBoxes; ++b) {
        const int row = __shfl_sync(0xffffffffu, rows, b);
        if (leader && b < boxes) {
#pragma unroll
          for (int c = 0; c < kHalves; ++c) tma_load_2d(to + b * box_bytes + c * (kKeys * kBoxDims * 2), &map_kv, c * kBoxDims, row, bar);
        }
      }
      rows = j + 1 < n ? look_up(j + 1) : 0;
    }
  } else if (warp < 4) {
    // S(u, j) = Q(u) . K(j)^T, as soon as the threads of row tile u have the scores before in registers; a warp per row tile.  The whole warp goes through the
    // loop and one lane issues, so that what the instructions take stays in uniform registers.
    constexpr uint32_t idesc = umma_instr_desc(kPairsTC, kKeys);
    constexpr uint32_t kQSub = (kPairsTC * kBoxDims * 2) >> 4, kKSub = (kKeys * kBoxDims * 2) >> 4;   // one sub-tile of 64 dims further, in descriptor units
    const int u = warp - 2, mine = u == 0 ? n0 : n1;
    const uint32_t q_low = umma_desc_low(smem_u32(sm.q[u])), k_low = umma_desc_low(smem_u32(sm.k)), to = tmem + kScoreCol0 + u * kKeys;
    const bool leader = elect_one();
    RingPosition<kStages> ring;
    bool ok = mine == 0 || warp_wait(&sm.q_full, 0, gave_up);
    for (int j = 0; j < mine && ok; ++j, ring.advance()) {
      ok = warp_wait(&sm.k_full[ring.stage], ring.phase, gave_up);
      if (ok && j > 0) ok = warp_wait(&sm.s_read[u], (j - 1) & 1, gave_up);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const uint32_t k_tile = k_low + ring.stage * ((kKeys * D * 2) >> 4);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)   // 16 dims further: 32 bytes inside a sub-tile's rows, then the next sub-tile
          umma_bf16(to, q_low + (kk >> 2) * kQSub + (kk & 3) * 2, k_tile + (kk >> 2) * kKSub + (kk & 3) * 2, idesc, kk > 0 ? 1u : 0u);
        umma_commit(&sm.s_full[u]);
        umma_commit(&sm.k_empty[ring.stage]);
      }
    }
    for (int j = mine; j < n && ok; ++j, ring.advance()) {   // none of this tile's rows sees these keys
      ok = warp_wait(&sm.k_full[ring.stage], ring.phase, gave_up);
      if (ok && leader) mbar_arrive(&sm.k_empty[ring.stage]);
    }
  } else if (warp == 4) {
    // O(u) += P(u, j) . V(j) as soon as the weights are there
    constexpr uint32_t idesc = instr_desc_b_mn(kPairsTC, D);
    // V is the MN-major operand: beyond 64 dims the next sub-tile lies this far on, which the leading-dimension offset says; one sub-tile needs none
    constexpr uint32_t kVLeading = kHalves > 1 ? (kKeys * kBoxDims * 2) >> 4 : 1u;
    const uint32_t v_low = ((smem_u32(sm.v) >> 4) & 0x3FFF) | (kVLeading << 16);
    const bool leader = elect_one();
    RingPosition<kStages> ring;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j, ring.advance()) {
      ok = warp_wait(&sm.v_full[ring.stage], ring.phase, gave_up);
      const uint32_t v_tile = v_low + ring.stage * ((kKeys * D * 2) >> 4);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!ok || j >= (u == 0 ? n0 : n1)) continue;
        ok = warp_wait(&sm.p_full[u], j & 1, gave_up);
        if (!ok) continue;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)   // 16 keys further: 8 columns of P, 16 rows (2048 bytes) down in a V sub-tile
            umma_bf16_a_tmem(tmem + u * D, tmem + kWeightCol0 + u * kWeightCols + kk * 8, v_tile + kk * ((16 * kBoxDims * 2) >> 4), idesc, (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&sm.pv_done[u]);
        }
      }
      if (ok && leader) umma_commit(&sm.v_empty[ring.stage]);
    }
  } else if (warp >= kFirstSoftmaxWarp) {
    // (Two threads per pair, half of a tile's keys each and the maximum agreed on at a barrier, took 5 to 10 % longer.)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
    const int u = (warp - kFirstSoftmaxWarp) / 4, sub = warp & 3, pair = sub * 32 + lane, mine = u == 0 ? n0 : n1;
    const uint32_t lane_base = (uint32_t)(sub * 32) << 16;
    const uint32_t tmem_s = tmem + lane_base + kScoreCol0 + u * kKeys, tmem_p = tmem + lane_base + kWeightCol0 + u * kWeightCols, tmem_o = tmem + lane_base + u * D;
    const int tile_rows = max(0, min(tile_tokens, tokens - u * tile_tokens));
    const bool mine_valid = pair < tile_rows * group;
    const int token = token0 + u * tile_tokens + pair / group, head = kvh * group + pair % group;
    const int limit = mine_valid ? limit_of(token) : 0;
    if (!OWN) {
      const int fewest = __reduce_min_sync(0xffffffffu, mine_valid ? limit : kNoKey);
      if (lane == 0) atomicMin(&sm.lowest[u], fewest);
      tile_barrier(u);
    }
    const int lowest = sm.lowest[u];
    const float sl2 = p.scale * kToLog2;
    float reference = -INFINITY, row_sum = 0.0f;
    RingPosition<kStages> at;
    bool ok = true;   // (a warp that gives up goes on to the end without waiting: the others of its row tile meet it at their barriers)
    // Turn -1 works on whatever tensor memory holds and hands nothing on: the loop's instructions are fetched while the first keys are on their way (fetched behind them, the first
    // tile took 5,000 cycles where the others take 2,000).
    auto take_tile = [&](int j, auto some_masked) {
      constexpr bool masked = decltype(some_masked)::value;
      const int key0 = (kt_begin + max(j, 0)) * kKeys;
      if (j >= 0 && ok) ok = warp_wait(&sm.s_full[u], j & 1, gave_up);
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      float sc[kKeys];
      {
        uint32_t raw[kKeys];
#pragma unroll
        for (int c = 0; c < kKeys; c += 8) tmem_load_8(tmem_s + c, raw + c);
        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
        for (int i = 0; i < kKeys; ++i) sc[i] = __uint_as_float(raw[i]);
      }
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      if (lane == 0 && j >= 0) mbar_arrive(&sm.s_read[u]);   // (the load was warp-wide: every lane has its scores)
      if (masked) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) sc[i] = key0 + i < limit && (!JOINS || key0 + i >= p.first_key) ? sc[i] : -INFINITY;
      }
      float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
      for (int i = 0; i < kKeys; i += 8) {
        m0 = max3(m0, sc[i], sc[i + 1]);
        m1 = max3(m1, sc[i + 2], sc[i + 3]);
        m2 = max3(m2, sc[i + 4], sc[i + 5]);
        m3 = max3(m3, sc[i + 6], sc[i + 7]);
      }
      const float scaled_max = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * sl2;
      // The output and the sum are taken against a reference, which moves only where a tile's maximum is far above it (the first tile's always is).
      const bool grown = scaled_max > reference + kLazyRescale;
      if (__builtin_expect(__any_sync(0xffffffffu, grown), 0)) {
        if (j > 0) {
          if (ok) ok = warp_wait(&sm.pv_done[u], (j - 1) & 1, gave_up);   // the product that last added to the output
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const float alpha = grown ? exp2f(reference - scaled_max) : 1.0f;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {   // (loads and stores are warp-wide: rows that need nothing multiply by one)
            uint32_t o[16];
            tmem_load_16(tmem_o + c, o);
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_store_8(tmem_o + c, o);
            tmem_store_8(tmem_o + c + 8, o + 8);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
          row_sum *= alpha;
        }
        if (grown) reference = scaled_max;
      }
      const float base = reference == -INFINITY ? 0.0f : reference;   // a row that has seen no key yet: every weight is 0
      if (masked) {
        // Values of keys that none of the CTA's rows sees (never written, perhaps) become zeros: 0 * (whatever is there) must stay 0.  Of keys that some rows see, what is
        // not finite is taken out and noted.
        const bool some_see = lowest < min(key0 + kKeys, last);
        const int none_from = max(0, min(kKeys, last - key0)), none_to = JOINS ? max(0, min(kKeys, p.first_key - key0)) : 0;
        if (none_from < kKeys || none_to > 0 || some_see) {
          if (ok) ok = warp_wait(&sm.v_full[at.stage], at.phase, gave_up);
          uint8_t* v_tile = reinterpret_cast<uint8_t*>(sm.v[at.stage]);
          for (int r = pair >> 3; r < kKeys; r += kPairsTC / 8) {   // 8 threads a row of 128 bytes, whatever the swizzle
            if (r < none_to || r >= none_from) {
#pragma unroll
              for (int c = 0; c < kHalves; ++c) *reinterpret_cast<uint4*>(v_tile + c * (kKeys * kBoxDims * 2) + r * 128 + (pair & 7) * 16) = make_uint4(0, 0, 0, 0);
            } else if (some_see) {
#pragma unroll
              for (int c = 0; c < kHalves; ++c) {
                uint8_t* chunk = v_tile + c * (kKeys * kBoxDims * 2) + r * 128 + (pair & 7) * 16;
                const uint4 eight = *reinterpret_cast<const uint4*>(chunk);
                if (__builtin_expect(not_finite(eight.x) | not_finite(eight.y) | not_finite(eight.z) | not_finite(eight.w), 0u) != 0u)
                  take_out(reinterpret_cast<uint16_t*>(chunk), &sm.bad[0][c * kBoxDims + (((pair & 7) ^ (r & 7)) << 3)], D, key0 + r, &sm.any_bad);   // the 128-byte swizzle: chunk i of row r lies at i ^ (r % 8)
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // generic-proxy writes -> visible to the tensor core
        }
      }
      // The warps of the two row tiles that share a scheduler take turns: one's exponentials, which the exponential unit sets the pace of, run under the other's loads, maxima and
      // stores.  Left alone they fall into step and wait for the unit together, then leave it idle together (2,750 cycles a tile).
      if (ok && (u == 0 ? j > 0 && j <= n1 : j >= 0 && j < n0)) ok = warp_wait(&sm.exps_done[u ^ 1][sub], (u == 0 ? j - 1 : j) & 1, gave_up);
      const Pair scale2 = pair_of(sl2, sl2), minus_base2 = pair_of(-base, -base);
      Pair sums = pair_of(0.0f, 0.0f);
      uint32_t packed[kKeys / 2];
#pragma unroll
      for (int i = 0; i < kKeys / 2; ++i) {
        float x0, x1;
        unpair(fma2(pair_of(sc[2 * i], sc[2 * i + 1]), scale2, minus_base2), x0, x1);
        const float p0 = exp2_approx(x0), p1 = exp2_approx(x1);
        sums = add2(sums, pair_of(p0, p1));
        // A weight keeps 8 bits where it meets its value, as in the other bfloat16 attention kernels (the product takes bfloat16); the sum has all of it.  Over some thousand keys
        // that is an error of 1.6e-3 of the output, as much as the output's own rounding.
        packed[i] = pack_bf16(p0, p1);
      }
      if (lane == 0 && j >= 0) mbar_arrive(&sm.exps_done[u][sub]);
      if (j > 0 && ok) ok = warp_wait(&sm.pv_done[u], (j - 1) & 1, gave_up);   // the weights before have been read
#pragma unroll
      for (int c = 0; c < kKeys / 2; c += 4) tmem_store_4(tmem_p + c, packed + c);
      asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      __syncwarp();
      if (lane == 0 && j >= 0) mbar_arrive(&sm.p_full[u]);
      float sum0, sum1;
      unpair(sums, sum0, sum1);
      row_sum += sum0 + sum1;
      if (j >= 0) {
        at.advance();
      } else {
        reference = -INFINITY;
        row_sum = 0.0f;
      }
    };
    // Tiles that every row sees all of, then the others: what the masks take stays out of the loop that counts (with it inside, every tile took a fifth longer).  Own keys behind a prefix that
    // ends inside a tile all go through the other loop, for their first tile's sake.
    const int all_seen = JOINS && p.first_key % kKeys != 0 ? 0 : max(0, min(mine, lowest / kKeys - kt_begin));
    int j = -1;
    for (; mine > 0 && j < all_seen; ++j) take_tile(j, std::false_type{});
    for (; mine > 0 && j < mine; ++j) take_tile(j, std::true_type{});
    if (ok && mine > 0) ok = warp_wait(&sm.pv_done[u], (mine - 1) & 1, gave_up);
    // Where only the other row tile has keys (a portion that begins inside the prefix), this one's queries are copied too, and nothing above has waited for them: they land
    // before anything else is put in their place.
    if (JOINS && mine == 0 && n > 0) ok = warp_wait(&sm.q_full, 0, gave_up);
    if (JOINS) grid_dependency_wait();   // the prefix's parts
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const size_t at_pair = (size_t)token * p.q_heads + head;
      const bool any_bad = *(volatile int*)&sm.any_bad != 0;
      float top = reference, total = row_sum, factor = 1.0f;
      float4* staged = reinterpret_cast<float4*>(sm.q[u]) + sub * 32 * 4;
      float* factors = reinterpret_cast<float*>(sm.q[u]) + kPairsTC * 16 + sub * 32 * kOwnParts<D>;   // [part][the warp's row]
      if (JOINS) {
        const float2* parts_ml = p.part_ml + at_pair * p.parts;
#pragma unroll 2
        for (int i = 0; i < p.parts; ++i) top = fmaxf(top, mine_valid ? __ldcg(parts_ml + i).x : -INFINITY);
        factor = reference == -INFINITY ? (row_sum == 0.0f ? 0.0f : 1.0f) : exp2f(reference - top);   // (a part of nothing but NaN keeps its NaN)
        total = row_sum * factor;
#pragma unroll 2
        for (int i = 0; i < p.parts; ++i) {
          const float2 ml = mine_valid ? __ldcg(parts_ml + i) : make_float2(-INFINITY, 0.0f);
          const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2f(ml.x - top);
          if (f != 0.0f) total = fmaf(f, ml.y, total);
          factors[i * 32 + lane] = f;
        }
      } else if (!OWN && mine_valid) {
        p.part_ml[at_pair * p.parts + blockIdx.x] = make_float2(reference, row_sum);
      }
      const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
      // A thread has its row, memory wants lines: 16 columns of the warp's 32 rows go through shared memory (Q's place: it has landed and its products are done, or it was never
      // copied), piece i of row r at i ^ (r / 2 % 4).
      // Row r = 8 i + lane / 4, piece lane % 4, is then a lane's i-th, of the prefix's parts too.  (Without parts a thread writes its own row: 32 bytes at a time, and less code to fetch.)
      const int quarter = lane & 3;
      size_t pair_at[4];
      bool there[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int other = sub * 32 + 8 * i + (lane >> 2);
        there[i] = other < tile_rows * group;
        pair_at[i] = (size_t)(token0 + u * tile_tokens + other / group) * p.q_heads + kvh * group + other % group;
      }
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {   // (the load is warp-wide: every lane takes part)
        uint32_t raw[16];
        if (mine > 0) {
          tmem_load_16(tmem_o + c, raw);
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
        }
        float o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = mine > 0 ? __uint_as_float(raw[i]) : 0.0f;
        if (__builtin_expect(any_bad, 0)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const volatile int* first = &sm.bad[0][c + i];
            const bool plus = first[0] < limit, minus = first[D] < limit, none = first[2 * D] < limit;
            if (none || (plus && minus)) o[i] = __int_as_float(0x7fffffff);
            else if (plus) o[i] += INFINITY;
            else if (minus) o[i] -= INFINITY;
          }
        }
        if (!OWN && mine <= 0) continue;
        if (OWN) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = JOINS && factor == 0.0f ? 0.0f : o[i] * factor;
          if (!JOINS) {
            uint4* to = reinterpret_cast<uint4*>(p.out + at_pair * D + c);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (mine_valid)
                to[i] = make_uint4(pack_bf16(o[8 * i] * inverse, o[8 * i + 1] * inverse), pack_bf16(o[8 * i + 2] * inverse, o[8 * i + 3] * inverse),
                                   pack_bf16(o[8 * i + 4] * inverse, o[8 * i + 5] * inverse), pack_bf16(o[8 * i + 6] * inverse, o[8 * i + 7] * inverse));
            continue;
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) staged[lane * 4 + (i ^ ((lane >> 1) & 3))] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
        float4 sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2);
          sums[i] = staged[r * 4 + (quarter ^ ((r >> 1) & 3))];
          if (!OWN && there[i]) reinterpret_cast<float4*>(p.part_o + (pair_at[i] * p.parts + blockIdx.x) * D + c)[quarter] = sums[i];
        }
        if (OWN) {
#pragma unroll 2
          for (int part = 0; part < p.parts; ++part) {
            float4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = there[i] ? __ldcg(reinterpret_cast<const float4*>(p.part_o + (pair_at[i] * p.parts + part) * D + c) + quarter) : sums[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float f = factors[part * 32 + 8 * i + (lane >> 2)];
              if (f != 0.0f)   // (a part without keys was not written)
                sums[i].x = fmaf(f, v[i].x, sums[i].x), sums[i].y = fmaf(f, v[i].y, sums[i].y), sums[i].z = fmaf(f, v[i].z, sums[i].z), sums[i].w = fmaf(f, v[i].w, sums[i].w);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float by = __shfl_sync(0xffffffffu, inverse, 8 * i + (lane >> 2));
            if (there[i])
              reinterpret_cast<uint2*>(p.out + pair_at[i] * D + c)[quarter] = make_uint2(pack_bf16(sums[i].x * by, sums[i].y * by), pack_bf16(sums[i].z * by, sums[i].w * by));
          }
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  }
  close_and_report(gave_up, p.error_flag);
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

template <int D, bool OWN, bool JOINS>
static int launch_tc(const CUtensorMap& map_q, const CUtensorMap& map_kv, const PrefixTCParams& p, dim3 grid, cudaStream_t stream) {
  static std::atomic<unsigned long long> devices{0};
  static std::atomic<int> registers{0};
  const int smem = (int)sizeof(SmemPrefix<D>) + 1024;
  static_assert(sizeof(SmemPrefix<D>) + 1024 <= 232448, "shared memory of a CTA");
  cudaError_t e = allow_shared_memory(prefix_tc_kernel<D, OWN, JOINS>, smem, devices);
  if (e != cudaSuccess) return (int)e;
  if (registers.load(std::memory_order_relaxed) == 0) {   // the warps' shares are handed out of what the launch holds: less than that would wait for good
    cudaFuncAttributes found;
    e = cudaFuncGetAttributes(&found, prefix_tc_kernel<D, OWN, JOINS>);
    if (e != cudaSuccess) return (int)e;
    registers.store(found.numRegs, std::memory_order_relaxed);
  }
  if (registers.load(std::memory_order_relaxed) < kLaunchRegs) return (int)cudaErrorLaunchOutOfResources;
  return (int)launch_pdl(prefix_tc_kernel<D, OWN, JOINS>, grid, dim3(kThreadsTC), (size_t)smem, stream, map_q, map_kv, p);
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
  if (own && (parts > (head_dim == 64 ? kOwnParts<64> : kOwnParts<128>) || (parts > 0) != (first_key > 0))) return (int)cudaErrorInvalidValue;
  if (kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > kPairsTC || kv_heads > 65535 || page_size <= 0 || page_size % 16 != 0 || num_pages <= 0 || q_row_stride % 8 != 0 ||
      (head_dim != 64 && head_dim != 128) || error_flag == nullptr || ((uintptr_t)q & 15) || ((uintptr_t)pages & 15) || ((uintptr_t)out & 15) || ((uintptr_t)part_o & 15) ||
      ((uintptr_t)part_ml & 7) || (!own && (parts < 1 || shared < 1)))
    return (int)cudaErrorInvalidValue;
  const int group = q_heads / kv_heads, tile_tokens = kPairsTC / group;
  const long long pool_rows = (long long)num_pages * 2 * kv_heads * page_size;
  if (pool_rows >= 0x7fffffffLL - 256) return (int)cudaErrorInvalidValue;   // a copy's row is a 32-bit coordinate
  const int keys = head_dim == 64 ? kKeysOf<64> : kKeysOf<128>;
  int box_keys = 16;   // keys of a box: what divides a page and a key tile
  while (page_size % (2 * box_keys) == 0 && keys % (2 * box_keys) == 0) box_keys *= 2;
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
    if (parts > 0) return head_dim == 64 ? launch_tc<64, true, true>(map_q, map_kv, p, grid, stream) : launch_tc<128, true, true>(map_q, map_kv, p, grid, stream);
    return head_dim == 64 ? launch_tc<64, true, false>(map_q, map_kv, p, grid, stream) : launch_tc<128, true, false>(map_q, map_kv, p, grid, stream);
  }
  if (pieces > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid(parts, kv_heads, pieces);
  return head_dim == 64 ? launch_tc<64, false, false>(map_q, map_kv, p, grid, stream) : launch_tc<128, false, false>(map_q, map_kv, p, grid, stream);
}
