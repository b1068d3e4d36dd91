// Attention of drafted trees over the paged KV cache: the verification step of speculative
// decoding. Each sequence has a tree of T drafted nodes (packed end to end over the batch);
// node n's query attends to the sequence's cached keys 0 .. len - 1, read in place from its
// blocks, and to the nodes whose bit is set in its mask row (its ancestors and itself),
// whose K/V are given apart from the cache, so that nothing rejected is ever written there:
//   out[n, h] = sum_j p_j v_j,  p = softmax_j(scale * q[n, h] . k_j)
// A row that sees no key gives zeros. No counterpart in the reference, which decodes one
// token per sequence and step (engine/kv_cache.py:611-620).
//
// All of a tree's rows share the context keys, so K/V are streamed once for up to
// 128 / group nodes x group query heads: one tile of 128 MMA rows. What bounds it is that
// stream (2 * 2 * D bytes per key and KV head) up to a full tile, and the exponentials
// (one per row and key) for wider trees.
//
// Work split. Item = (sequence, KV head, tile of 128 rows), W = ceil(T / 64) + ceil(len / 64)
// stages of 64 keys (the tree's own first) plus a charge of kItemCost for its start and end.
// All items are laid end to end and cut into equal ranges, one per CTA, whatever the mix of
// lengths; every CTA derives the same ranges from the lengths on the device, so nothing of
// the plan needs the host to know one. An item inside one range writes its output; one cut
// between ranges leaves its pieces' states (running maximum, sum, unnormalised output, all
// float32; a range has at most two cut pieces, its first and its last), which the CTAs of those
// pieces join. Where every tree has the same number of tiles, the tiles of an item go to as many
// CTAs side by side over the same range of keys, so that they share its reads in L2 (bf16, 28 / 4
// heads of 128: 16 trees of 64 nodes over 16K keys 342 us, 382 with each tile an item of its own;
// 16 of 40 over 8K 137 and 145; 32 of 20 over 16K 338 either way).
//
// Inside a CTA: one warp issues the TMA copies of K, one those of V. The stages go in turn to
// two streams, each a warp that issues tcgen05 MMAs and four softmax warps (a row per
// thread) with two score buffers and an accumulator of its own in TMEM: S = Q K^T (128 x 64,
// float32), P = 2^(S - m) in the storage type over S, O += P V against a maximum m
// that moves only when a row's maximum grew by more than kSlack (in log2). The scores of a
// stream's next stage are made while its warps work on the present one's, and one stream
// computes exponentials while the other waits; their states are joined at the end of a piece.
// P goes to the tensor cores as in this package's other attention kernels: float16 keeps 11
// bits of a weight; bfloat16 keeps 8, so what that leaves of it follows as a second half (S leaves
// room for both) and V is multiplied by either. The row sum is taken in float32, before any of it.
//
// Measured (B200, captured calls): 16 trees of 9-18 nodes over 8K-32K keys, 28 / 4 heads of 128,
// bf16: 134 us = 4.9 TB/s, 0.76 of the copy bandwidth; 156-167 us for a lone call on a flushed
// L2. 64 trees of 1-26 nodes over 128-2048 keys, 14 / 2 heads of 64, fp16: 27.6 us (1.4 TB/s; an
// item has 3 to 33 stages, so starts, ends and the set-up weigh as much as its stages). 4 trees
// of 129-256 nodes over 1000-4100 keys, bf16: 60-65 us = 0.5 PFLOP/s, tensor cores busy 40 % of
// the time, exponentials 27 %. One tree of 8 nodes over 129 keys: 9 us, a launch, the plan, one
// load and one stage behind one another. What bounds the wide cases is the warps' own
// instructions, with three warps on a scheduler to hide their latency.
// The second halves of bfloat16's weights cost 123 -> 134 us, 56 -> 62 us, and 262 -> 342 us for
// 16 trees of 64 nodes over 16K keys, by their products and the softmax warps' arithmetic.
// Slower, measured before them (long case then 122-128 us): two softmax warps per row (142),
// stages of 128 keys with one score buffer (136), four streams at head_dim 64 (88-127 us for 77),
// a separate launch for the join (7-11 us more on short calls).
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace pkv {
namespace {

constexpr int kBS = 16;
constexpr int kNK = 64;          // keys per stage
constexpr int kStreams = 2;
constexpr int kRing = 4;         // stages of the K ring and of the V ring
constexpr int kBars = 4 * kRing + 3 * kStreams + 5;
constexpr int kMaxSeqs = 1024;   // sequences per call: their tables live in shared memory
constexpr int kMaxWords = 8;     // mask words of 64 nodes
// An item's start and end, in stages, and the least that a CTA gets, each as good as any on small
// and large calls. Charge 5: serving batch 29.5 us for 27.7; 11: 28.0, wide trees alike. Least 4:
// no different; 12: one tree over 16K keys 28.2 us for 25.2.
constexpr int kItemCost = 8;
constexpr int kMinRange = 8;
constexpr int kMaxPieces = 160;  // CTAs at most: an item's pieces
constexpr float kLog2e = 1.4426950408889634f;
// Every slot of a ring belongs to one stream, so that a wait sees each of its phases.
static_assert(kRing % (2 * kStreams) == 0, "ring slots per stream and score buffer");

template <int D> struct TreeShape {
  static constexpr int DC = D / 64;             // 64-wide head_dim chunks
  static constexpr int GB = DC * 1024;          // eight keys of K (or V): [DC][8 keys][64], 128B-swizzled
  static constexpr int KSB = kNK / 8 * GB;      // a stage of them
  static constexpr int QB = DC * 128 * 128;     // the Q tile: [DC][128 rows][64], 128B-swizzled
  // TMEM columns: two score buffers and an accumulator per stream.
  static constexpr int OCOL = kStreams * 2 * kNK;
  static constexpr int NCOLS = 512;
  static_assert(OCOL + kStreams * D <= NCOLS, "TMEM columns");
  static_assert(kMaxPieces * 128 * 4 <= 2 * QB + 2 * kRing * KSB, "the join's maxima");
  static constexpr int SW = 4 * kStreams;       // softmax warps
  static constexpr int THREADS = (SW + 2 + kStreams) * 32;
  static constexpr int SMEM = 1024 + 2 * QB + 2 * kRing * KSB + (kBars + 2) * 8 + 2 * kStreams * 2 * 128 * 4 +
                              5 * kMaxSeqs * 4;
};

// The CTAs' equal shares of all stages, as every CTA derives them from the lengths.
struct TreePlan {
  int ranges;     // CTAs (or gangs of them) that share the stages
  int gang;       // tiles side by side: a gang's CTAs; 1 = a tile is an item of its own
  int quota, rem; // range g: quota stages, one more if g < rem
  __device__ int start(int g) const { return g * quota + min(g, rem); }
  __device__ int range_of(int x) const;  // the range that holds position x
};

// A CTA's piece of an item that several ranges share, for the join.
struct CutPiece {
  int node, head, rows;    // the tile's first node, KV head, rows
  int pieces, index;       // of the item (0: no such piece); which of them this is
  int first;               // CTA of the first piece
};

struct TreeParams {
  void* out;
  const int32_t* cu;
  const int32_t* ctx;
  const uint64_t* mask;
  const int32_t* tables;
  const int32_t* seq_rows;
  int32_t* status;
  int32_t* counts;     // [CTAs][2] of the cut item that begins in a CTA's range: pieces stored, shares joined
  float* part_ml;      // [2 per CTA][2][128] running maximum and sum
  float4* part_o;      // [2 per CTA][D / 4][128 rows]: four columns of a row, so a warp moves 512 bytes at a time
  int64_t out_st, out_sh, table_stride, total_nodes;
  int32_t table_rows, table_cols, batch, hkv, group, tile_nodes, words, layer, nbt;
  int32_t out_vec16, max_nodes;
  float scale_log2;
};

__device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// a / b for 0 <= a, 0 < b: by the reciprocal with one correction where float32 holds a
// exactly (the quotient is off by one at most), a third of an integer division's latency.
__device__ inline int quotient(int a, int b) {
  if (a >= 1 << 22) return a / b;
  const int q = (int)__fdividef((float)a, (float)b), r = a - q * b;
  return q + (r >= b) - (r < 0);
}

// A load past L1 (kept in program order, but not waited for).
__device__ inline float ld_cg(const float* ptr) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(ptr));
  return v;
}
__device__ inline float4 ld_cg(const float4* ptr) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(ptr));
  return v;
}

// 4-D bulk tensor copy global -> shared (no multicast), completion on an mbarrier.
__device__ inline void tma_load_4d(void* smem_dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                   uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

__device__ inline int TreePlan::range_of(int x) const {
  const int big = rem * (quota + 1);
  return x < big ? quotient(x, quota + 1) : rem + quotient(x - big, quota);
}

// The lengths of sequence b, clamped to what the call's own sizes allow.
struct SeqLens {
  int first, nodes, ctx, row;  // nodes -1: its offsets fall
};
__device__ inline SeqLens seq_lens(const TreeParams& p, int b, int32_t* status) {
  SeqLens s;
  const int lo = p.cu[b], hi = p.cu[b + 1];
  const int n = p.ctx[b], row = p.seq_rows ? p.seq_rows[b] : b;
  const bool bad = lo < 0 || hi < lo || hi > p.total_nodes || hi - lo > p.max_nodes || n < 0 ||
             n > (int64_t)p.table_cols * kBS || row >= p.table_rows;
  s.first = (int)min((int64_t)max(lo, 0), p.total_nodes);
  s.nodes = hi < lo ? -1 : min(max((int)min((int64_t)hi, p.total_nodes) - s.first, 0), p.max_nodes);
  s.row = row;
  // A padding row has no cached keys.
  s.ctx = row < 0 || row >= p.table_rows ? 0 : (int)min((int64_t)max(n, 0), (int64_t)p.table_cols * kBS);
  if (bad) report(status, PKV_ERR_OUT_OF_RANGE);
  return s;
}
__device__ inline int tiles_of(const TreeParams& p, int nodes) {
  return nodes <= p.tile_nodes ? nodes > 0 : quotient(nodes + p.tile_nodes - 1, p.tile_nodes);
}
__device__ inline int item_cost(int nodes, int ctx) { return kItemCost + ceil_div(nodes, kNK) + ceil_div(ctx, kNK); }

template <typename T, int D>
__global__ void __launch_bounds__(TreeShape<D>::THREADS, 1)
    tree_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                const __grid_constant__ CUtensorMap nmap_k, const __grid_constant__ CUtensorMap nmap_v,
                const __grid_constant__ CUtensorMap qmap, const TreeParams p) {
  using S = TreeShape<D>;
  constexpr int DC = S::DC, SW = S::SW;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                     // [2][QB]
  uint8_t* sK = sQ + 2 * S::QB;           // [kRing][KSB]
  uint8_t* sV = sK + kRing * S::KSB;      // [kRing][KSB]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kRing * S::KSB);
  uint64_t* k_full = bars;                // [kRing] K landed
  uint64_t* v_full = k_full + kRing;      // [kRing] V landed
  uint64_t* s_done = v_full + kRing;      // [kRing] S(j) = Q K(j)^T done: S ready, K slot free
  uint64_t* o_done = s_done + kRing;      // [kRing] O += P(j) V(j) done: V slot and score buffer free
  uint64_t* p_full = o_done + kRing;      // [kStreams][2] P stored, by score buffer
  uint64_t* o_free = p_full + 2 * kStreams;  // [kStreams] accumulators read, for a stream with stages in the piece
  uint64_t* q_full = o_free + kStreams;   // [2] Q landed, pieces in turn
  uint64_t* q_free = q_full + 2;          // [2] the piece's every MMA done
  uint64_t* mma_done = q_free + 2;        // every MMA of the CTA completed
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + kBars);
  float* s_ml = reinterpret_cast<float*>(bars + kBars + 2);  // [2 parities][kStreams][2][128] maxima and sums
  int32_t* s_off = reinterpret_cast<int32_t*>(s_ml + 2 * kStreams * 2 * 128);  // [batch] where its items begin
  int32_t* s_first = s_off + kMaxSeqs;                                         // [batch] first node
  int32_t* s_nodes = s_first + kMaxSeqs;                                       // [batch] nodes
  int32_t* s_ctx = s_nodes + kMaxSeqs;                                         // [batch] cached keys
  int32_t* s_row = s_ctx + kMaxSeqs;                                           // [batch] table row
  __shared__ CutPiece s_cut[2];  // this range's cut pieces: one that began before it, one that ends behind it
  __shared__ int s_joins[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = p.batch, G = p.group;

  // Set-up by warps that have no lengths to read in a small batch.
  if (warp == SW && lane == 0) {
    s_cut[0].pieces = s_cut[1].pieces = 0;
    for (int i = 0; i < 4 * kRing; ++i) mbar_init(&bars[i], 1);
    for (int i = 0; i < 2 * kStreams; ++i) mbar_init(&p_full[i], 4);
    for (int i = 0; i < kStreams; ++i) mbar_init(&o_free[i], SW);
    for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 1), mbar_init(&q_free[i], 1);
    mbar_init(mma_done, kStreams);
    fence_mbar_init();
  }
  if (warp == SW - 1) {
    tmem_alloc(tslot, S::NCOLS);
    tc_fence_before_sync();
  }
  if (warp == SW + 1 && lane == 0) {
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
    prefetch_tensormap(&nmap_k);
    prefetch_tensormap(&nmap_v);
    prefetch_tensormap(&qmap);
  }
  // ------------------------------------------------------------------ plan
  for (int b = tid; b < B; b += S::THREADS) {
    const SeqLens s = seq_lens(p, b, blockIdx.x == 0 ? p.status : nullptr);
    s_first[b] = s.first;
    s_nodes[b] = s.nodes;
    s_ctx[b] = s.ctx;
    s_row[b] = s.row;
  }
  __syncthreads();
  tc_fence_after_sync();
  // The rest by every warp for itself: no further barrier, and all write the same offsets.
  TreePlan plan;
  {
    const int per = ceil_div(B, 32), b0 = min(B, lane * per), b1 = min(B, b0 + per);
    constexpr int kDisorder = 1 << 30;
    int least = 1 << 30, most = 0, alone = 0, ganged = 0;  // stages if a tile is an item; if its item's tiles go together
    for (int b = b0; b < b1; ++b) {
      const int n = s_nodes[b];
      if (n < 0) most = kDisorder;
      if (n <= 0) continue;
      const int tiles = tiles_of(p, n), cost = p.hkv * item_cost(n, s_ctx[b]);
      least = min(least, tiles);
      most = max(most, tiles);
      alone += tiles * cost;
      ganged += cost;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    plan.gang = least == most && most > 1 && most <= (int)gridDim.x ? most : 1;
    const int mine = plan.gang > 1 ? ganged : alone;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    // Node offsets out of order (reported) would let trees overlap, and the sum of their stages pass
    // what the host has bounded by the nodes: then nothing is computed.
    const int total = most == kDisorder ? 0 : __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    for (int b = b0; b < b1; ++b) {
      s_off[b] = before;
      const int n = s_nodes[b];
      if (n > 0) before += p.hkv * (plan.gang > 1 ? 1 : tiles_of(p, n)) * item_cost(n, s_ctx[b]);
    }
    plan.ranges = max(1, min(quotient(gridDim.x, plan.gang), total / kMinRange));
    plan.quota = quotient(total, plan.ranges);
    plan.rem = total - plan.quota * plan.ranges;
    __syncwarp();
  }
  const uint32_t tmem = *tslot;
  uint64_t deadline = global_ns() + kWaitBudgetNs;  // per piece: a long call is no hang
  const int range = quotient(blockIdx.x, plan.gang), member = blockIdx.x - range * plan.gang;
  const int pos0 = range < plan.ranges ? plan.start(range) : 0;
  const int pos_end = range < plan.ranges ? plan.start(range + 1) : 0;

  // Every role walks the same pieces and numbers stages across them, so ring slots and
  // barrier parities continue from one piece to the next.
  struct Piece {
    int b, head, tile, rows, nodes, ctx, nns;  // nns: the item's stages of the tree's own keys, its first
    int s0, nst, item_end;                     // first stage, stages; position behind the item
    bool begins, ends;
  };
  auto next_piece = [&](int& pos, Piece& u) -> bool {
    while (pos < pos_end) {
      int lo = 0, hi = B - 1;  // the last sequence that begins at or before pos (empty ones take no room)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_off[mid] <= pos) lo = mid; else hi = mid - 1;
      }
      u.b = lo;
      u.nodes = s_nodes[lo];
      u.ctx = s_ctx[lo];
      const int cost = item_cost(u.nodes, u.ctx), tiles = plan.gang > 1 ? 1 : tiles_of(p, u.nodes);
      const int rel = pos - s_off[lo], item = quotient(rel, cost), x0 = rel - item * cost;
      const int x1 = min(cost, x0 + (pos_end - pos)), item_end = pos + cost - x0;
      pos += x1 - x0;
      u.s0 = max(0, x0 - kItemCost);
      u.nst = max(0, x1 - kItemCost) - u.s0;
      if (u.nst <= 0) continue;
      u.head = tiles == 1 ? item : quotient(item, tiles);
      u.tile = plan.gang > 1 ? member : item - u.head * tiles;
      u.rows = min(p.tile_nodes, u.nodes - u.tile * p.tile_nodes) * G;
      u.nns = ceil_div(u.nodes, kNK);
      u.begins = u.s0 == 0;
      u.ends = x1 == cost;
      u.item_end = item_end;
      deadline = global_ns() + kWaitBudgetNs;
      return true;
    }
    return false;
  };
  auto first_of = [](int stream, int gs) { return (stream + kStreams - gs % kStreams) % kStreams; };  // its first stage

  // Registers: the copy and MMA warps (one warpgroup) hand most of theirs to the softmax
  // warps. 256 x 224 + 128 x 56 = 384 x 168, what the launch got.
  static_assert(S::THREADS == 384 && SW == 8, "register split");
  if (warp >= SW) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp < SW + 2) {
    // ---------------------------------------------------------------- TMA copies: a warp for K, one for V
    // What these warps cost per stage sets the pace of the whole CTA (measured at head_dim 128,
    // in cycles: waits that find their barrier complete 180, a copy 85 to 110 whichever lane
    // issues it, the loop's own arithmetic 450), so a block's keys are one copy (the layout in
    // shared memory takes groups of 8 keys, all of a row's chunks) and the loops over the tree's
    // own keys and the context's are apart. (Before bfloat16's weights had second halves: two copies
    // a block and one loop 128 us for 16 trees of 40 nodes over 8K keys, so 118; four copy warps
    // 113-118 where two took 107, for the registers and issue slots they take from the softmax
    // warps.)
    const bool is_v = warp != SW;
    uint8_t* const ring = is_v ? sV : sK;
    uint64_t* const full = is_v ? v_full : k_full;
    uint64_t* const done = is_v ? o_done : s_done;  // the slot's last reader
    const CUtensorMap* const cmap = is_v ? &tmap_v : &tmap_k;
    const CUtensorMap* const nmap = is_v ? &nmap_v : &nmap_k;
    bool ok = true;
    int gs = 0, k = 0, stopped = 0;  // stages and pieces before this one; the stage a wait ran out at
    Piece u;
    for (int pos = pos0; ok && next_piece(pos, u); gs += u.nst, ++k) {
      const int32_t* table = u.ctx > 0 ? p.tables + (int64_t)s_row[u.b] * p.table_stride : nullptr;
      const int nkb = ceil_div(u.ctx, kBS);
      const int own = max(0, u.nns - u.s0);  // leading stages of the tree's own keys
      const int own_end = min(own, u.nst);
      const int kb0 = max(0, u.s0 - u.nns) * (kNK / kBS);
      // The first of a block's groups of keys in the pool's tensor map; for blocks past the
      // sequence, which are not copied, any will do.
      auto lookup = [&](int kb) -> int {
        int blk = kb < nkb ? table[kb] : 0;
        if (blk < 0 || blk >= p.nbt) {
          report(p.status, PKV_ERR_OUT_OF_RANGE);
          blk = 0;
        }
        return ((p.layer * p.nbt + blk) * p.hkv + u.head) * (kBS / 8);
      };
      constexpr int kBlocks = kNK / kBS, kPerWindow = 32 / kBlocks;  // stages per window of 32 block ids
      int win = lookup(kb0 + lane), win_next = lookup(kb0 + 32 + lane);
      if (!is_v) {  // the piece's Q: rows (node, head of the group), those past the tree unused
        if (k >= 2) ok = mbar_wait_until(&q_free[k & 1], ((k >> 1) - 1) & 1, deadline);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          stopped = gs;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&q_full[k & 1], DC * 128 * G * p.tile_nodes);
        __syncwarp();
        if (lane < DC)
          tma_load_4d(sQ + (k & 1) * S::QB + lane * 128 * 128, &qmap, 0, lane, u.head * G,
                      s_first[u.b] + u.tile * p.tile_nodes, &q_full[k & 1]);
      }
      // Keys past the tree or the sequence come only as far as their group or block reaches: what
      // a slot holds there is masked (K) or cleared (V) by the softmax warps.
      for (int i = 0; i < own_end && ok; ++i) {
        const int j = gs + i, st = j % kRing;
        if (j >= kRing) ok = mbar_wait_until(&done[st], ((j / kRing) - 1) & 1, deadline);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          stopped = j;
          break;
        }
        const int node0 = (u.s0 + i) * kNK, copies = min(kNK / 8, ceil_div(u.nodes - node0, 8));
        if (lane == 0) mbar_arrive_expect_tx(&full[st], copies * S::GB);
        __syncwarp();
        if (lane < copies)
          tma_load_4d(ring + st * S::KSB + lane * S::GB, nmap, 0, s_first[u.b] + node0 + lane * 8, 0, u.head, &full[st]);
      }
      for (int i = own_end; i < u.nst && ok; ++i) {
        const int ci = i - own;  // context stage of the piece
        if (ci > 0 && ci % kPerWindow == 0) {
          win = win_next;
          win_next = lookup(kb0 + 32 * (ci / kPerWindow + 1) + lane);
        }
        const int group = __shfl_sync(0xffffffffu, win, (ci * kBlocks + lane) % 32);
        const int j = gs + i, st = j % kRing;
        if (j >= kRing) ok = mbar_wait_until(&done[st], ((j / kRing) - 1) & 1, deadline);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          stopped = j;
          break;
        }
        const int copies = min(kBlocks, nkb - kb0 - ci * kBlocks);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], copies * (kBS / 8) * S::GB);
        __syncwarp();
        if (lane < copies) tma_load_4d(ring + st * S::KSB + lane * (kBS / 8) * S::GB, cmap, 0, 0, 0, group, &full[st]);
      }
    }
    if (!ok && lane == 0) report(p.status, PKV_ERR_TIMEOUT);
    // No copy may still be under way when the CTA leaves its shared memory. The MMA warps wait for
    // each of them, unless one gave up: so every ring slot's last copy, and every Q buffer's, again.
    const int issued = ok ? gs : stopped;
    const uint64_t until = global_ns() + kWaitBudgetNs;
    for (int j = max(0, issued - kRing); j < issued; ++j) mbar_wait_until(&full[j % kRing], (j / kRing) & 1, until);
    for (int x = max(0, k - 2); x < k && !is_v; ++x) mbar_wait_until(&q_full[x & 1], (x >> 1) & 1, until);
  } else {
    // ---------------------------------------------------------------- MMA issue, one warp per stream
    if (lane == 0) {
      const int stream = warp - SW - 2;
      constexpr bool kBf16 = Dt<T>::code == PKV_BF16;
      constexpr uint32_t idesc_s = umma_idesc_f16(kBf16, false, 128, kNK);
      constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, true, 128, D);
      const uint32_t to = tmem + S::OCOL + stream * D;
      auto ts_of = [&](int j) { return tmem + (stream * 2 + j / kStreams % 2) * kNK; };  // S(j), then P(j)
      // Shared memory ends below 2^18 bytes: a descriptor's address field takes offsets (in 16
      // bytes) by addition.
      const uint64_t dq = umma_desc_sw128(smem_u32(sQ), 16, 1024), dk = umma_desc_sw128(smem_u32(sK), 16, S::GB);
      const uint64_t dv = umma_desc_sw128(smem_u32(sV), 1024, S::GB);
      auto issue_s = [&](int j, int k) -> bool {  // of piece k
        const int st = j % kRing;
        const uint64_t aq = dq + (k & 1) * (S::QB / 16), bk = dk + st * (S::KSB / 16);
        if (!mbar_wait_until(&k_full[st], (j / kRing) & 1, deadline)) return false;
        const int jb = j - 2 * kStreams;  // whose P the score buffer holds, until its O has read it
        if (jb >= 0 && !mbar_wait_until(&o_done[jb % kRing], (jb / kRing) & 1, deadline)) return false;
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) 
          umma_f16_ss(ts_of(j), aq + (kk / 4 * 128 * 128 + kk % 4 * 32) / 16, bk + (kk / 4 * 1024 + kk % 4 * 32) / 16,
                      idesc_s, kk > 0);
        umma_commit(&s_done[st]);
        return true;
      };
      auto issue_o = [&](int j, bool first) -> bool {
        const int st = j % kRing;
        const uint64_t bv = dv + st * (S::KSB / 16);
        if (!mbar_wait_until(&v_full[st], (j / kRing) & 1, deadline)) return false;
        if (!mbar_wait_until(&p_full[stream * 2 + j / kStreams % 2], (j / (2 * kStreams)) & 1, deadline)) return false;
        tc_fence_after_sync();
#pragma unroll
        for (int kb = 0; kb < kNK / 16; ++kb) umma_f16_ts(to, ts_of(j) + kb * 8, bv + kb * 2 * S::GB / 16, idesc_o, !first || kb > 0);
        if constexpr (!Dt<T>::kExactP) {  // the weights' lo halves
#pragma unroll
          for (int kb = 0; kb < kNK / 16; ++kb)
            umma_f16_ts(to, ts_of(j) + kNK / 2 + kb * 8, bv + kb * 2 * S::GB / 16, idesc_o, true);
        }
        umma_commit(&o_done[st]);
        return true;
      };
      // A piece's first scores are made while the softmax warps still finish the one before;
      // only its first O waits until they have read the accumulators.
      bool ok = true;
      int gs = 0, k = 0, mine = 0;
      Piece u;
      for (int pos = pos0; ok && next_piece(pos, u); gs += u.nst, ++k) {
        const int i0 = first_of(stream, gs);
        if (i0 >= u.nst) continue;
        ok = mbar_wait_until(&q_full[k & 1], (k >> 1) & 1, deadline) && issue_s(gs + i0, k) &&
             (i0 + kStreams >= u.nst || issue_s(gs + i0 + kStreams, k)) &&
             (mine == 0 || mbar_wait_until(&o_free[stream], (mine - 1) & 1, deadline));
        for (int i = i0; i < u.nst && ok; i += kStreams)
          ok = issue_o(gs + i, i == i0) && (i + 2 * kStreams >= u.nst || issue_s(gs + i + 2 * kStreams, k));
        ++mine;
      }
      k = mine;
      if (!ok) report(p.status, PKV_ERR_TIMEOUT);
      if (k > 0) umma_commit(mma_done); else mbar_arrive(mma_done);
    }
  }
  } else {
    // ---------------------------------------------------------------- softmax warps
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int stream = warp / 4;
    const int r = (warp % 4) * 32 + lane;  // TMEM lane = tile row
    const int t = r / G, gq = r - t * G;   // node of the tile, query head of the group
    const uint32_t tl = tmem + ((uint32_t)((warp % 4) * 32) << 16);
    const uint32_t to = tl + S::OCOL + stream * D;
    // 2^(S - m) is at most 2^kSlack. In float16 it is made 2^kRaise times as large (so are the row
    // sums, and it leaves the output again with them): weights down to 2^-25 of m's are normal
    // numbers with all their bits and the largest are 2^15; unraised, a long tail beside one
    // dominant key would lose its bits from 2^-14 down and vanish below 2^-25.
    constexpr float kSlack = Dt<T>::kExactP ? 4.f : 8.f, kRaise = Dt<T>::kExactP ? 11.f : 0.f;
    bool ok = true;
    auto confirm = [&](int j) {  // O += P(j) V(j) has completed
      if (ok && !mbar_wait_until(&o_done[j % kRing], (j / kRing) & 1, deadline)) ok = false;
    };
    int gs = 0, k = 0, pos = pos0;
    Piece u, ahead;
    // The mask words of a piece's stage, loaded a stage ahead: the tree's own keys that this
    // row may see, and those that the lane's share of the tile's nodes may.
    uint64_t see_next = 0, any_next = 0;
    auto fetch_masks = [&](const Piece& x, int stage) {
      see_next = any_next = 0;
      if (stage >= x.nns) return;
      const int node0 = x.tile * p.tile_nodes;
      const uint64_t* const words = p.mask + ((int64_t)s_first[x.b] + node0) * p.words + stage;
      if (r < x.rows) see_next = words[(int64_t)t * p.words];
      for (int y = lane; y < min(p.tile_nodes, x.nodes - node0); y += 32) any_next |= words[(int64_t)y * p.words];
    };
    bool more = next_piece(pos, u);
    if (more) fetch_masks(u, u.s0 + first_of(stream, 0));
    for (; more; gs += u.nst, ++k, u = ahead) {
      const bool valid = r < u.rows;
      const bool live = (warp % 4) * 32 < u.rows;  // some row of the warp has a query
      const int64_t node = (int64_t)s_first[u.b] + u.tile * p.tile_nodes + t;

      float m = -INFINITY, l = 0.f;
      const int i0 = first_of(stream, gs);
      // Stage i of the piece: of the tree's own keys, or of the context's, whole or not. The three
      // are apart because every instruction of the loop counts (64 trees over 8K keys at head_dim
      // 64: 75 us in one loop, 71 so).
      auto step = [&](int i, auto own_keys, auto whole) {
        constexpr bool own = decltype(own_keys)::value;
        const int j = gs + i, sg = u.s0 + i, st = j % kRing;
        const int keys = own ? u.nodes - sg * kNK : u.ctx - (sg - u.nns) * kNK;  // of the stage, if < kNK
        const int buf = j / kStreams % 2;
        const uint32_t ts = tl + (stream * 2 + buf) * kNK;
        const bool partial = own || !decltype(whole)::value;  // not every row sees all of the stage's keys
        uint64_t see = ~0ull, seen = ~0ull;      // by this row, by any of the tile's
        if (partial) {
          if (own) {
            see = see_next;
            seen = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(any_next >> 32)) << 32 |
                   __reduce_or_sync(0xffffffffu, (uint32_t)any_next);
            if (i + kStreams < u.nst) fetch_masks(u, sg + kStreams);
          }
          if (keys < kNK) {
            see &= (1ull << keys) - 1;
            seen &= (1ull << keys) - 1;
          }
        }
        if (ok && !mbar_wait_until(&s_done[st], (j / kRing) & 1, deadline)) ok = false;
        tc_fence_after_sync();
        // Rows of V past the sequence or the tree, and those of nodes that no row sees (a padded
        // tree's), hold whatever was there, infinities and NaN included: 0 x NaN would reach the
        // output, so they are cleared in place.
        if (partial && seen != ~0ull) {
          if (ok && !mbar_wait_until(&v_full[st], (j / kRing) & 1, deadline)) ok = false;
          for (int x = r; x < kNK * DC * 8; x += 128) {
            const int key = x / (DC * 8);
            if (!((seen >> key) & 1))
              *reinterpret_cast<uint4*>(sV + st * S::KSB + key / 8 * S::GB + x / 8 % DC * 1024 + key % 8 * 128 + x % 8 * 16) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        if (live) {
          uint32_t sa[kNK];
#pragma unroll
          for (int c = 0; c < kNK / 32; ++c) tmem_ld32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sa + c * 32));
          tmem_wait_ld();
          if (partial) {
            const uint32_t lo32 = (uint32_t)see, hi32 = (uint32_t)(see >> 32);
#pragma unroll
            for (int e = 0; e < kNK; ++e)
              if (!(((e < 32 ? lo32 : hi32) >> (e & 31)) & 1)) sa[e] = __float_as_uint(-INFINITY);
          }
          float mt[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) mt[e] = fmaxf(__uint_as_float(sa[e]), __uint_as_float(sa[e + 4]));
#pragma unroll
          for (int e = 8; e < kNK; e += 8) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              mt[x] = fmaxf(fmaxf(mt[x], __uint_as_float(sa[e + x])), __uint_as_float(sa[e + 4 + x]));
          }
          const float mx = fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3])) * p.scale_log2;
          const float m_cand = fmaxf(m, mx);
          float alpha = 1.f;
          if (m_cand - m > kSlack) {  // false while both are -inf
            alpha = ex2(m - m_cand);
            m = m_cand;
            l *= alpha;
          }
          if (i > i0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            confirm(j - kStreams);
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t ob[32];
              tmem_ld32(to + c * 32, ob);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) ob[e] = __float_as_uint(__uint_as_float(ob[e]) * alpha);
              tmem_st32(to + c * 32, ob);
            }
          }
          const float mref = m == -INFINITY ? 0.f : m;
          float2 lsum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), negm2 = make_float2(kRaise - mref, kRaise - mref);
          tc_fence_after_sync();
#pragma unroll
          for (int c = 0; c < kNK / 32; ++c) {
            uint32_t pk[16], pl[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 x = ffma2(make_float2(__uint_as_float(sa[c * 32 + e]), __uint_as_float(sa[c * 32 + e + 1])), scale2,
                                     negm2);
              const float p0 = ex2(x.x), p1 = ex2(x.y);
              if constexpr (Dt<T>::kExactP) {
                pk[e / 2] = Dt<T>::pack(p0, p1);
              } else {
                // Cut, not rounded: what is left is below 2^-7 of the weight and the second half holds it
                // to 2^-8 of itself, 2^-15 in all, and cutting takes one instruction less.
                const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
                pk[e / 2] = __byte_perm(b0, b1, 0x7632);
                const float2 rest = ffma2(make_float2(__uint_as_float(b0 & 0xffff0000u), __uint_as_float(b1 & 0xffff0000u)),
                                          make_float2(-1.f, -1.f), make_float2(p0, p1));
                pl[e / 2] = Dt<T>::pack(rest.x, rest.y);
              }
              lsum[(e / 2) % 2] = fadd2(lsum[(e / 2) % 2], make_float2(p0, p1));
            }
            tmem_st16(ts + c * 16, pk);
            if constexpr (!Dt<T>::kExactP) tmem_st16(ts + kNK / 2 + c * 16, pl);
          }
          tmem_wait_st();
          l += (lsum[0].x + lsum[1].x) + (lsum[0].y + lsum[1].y);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[stream * 2 + buf]);
      };
      int i = i0;
      for (; i < u.nst && u.s0 + i < u.nns; i += kStreams) step(i, std::true_type{}, std::false_type{});
      const int full = min(u.nst, u.nns - u.s0 + u.ctx / kNK);  // stages before one that the sequence does not fill
      for (; i < full; i += kStreams) step(i, std::false_type{}, std::true_type{});
      if (i < u.nst) step(i, std::false_type{}, std::false_type{});
      more = next_piece(pos, ahead);
      if (more) fetch_masks(ahead, ahead.s0 + first_of(stream, gs + u.nst));
      // An item of two pieces is finished by the CTA of the first, at the end of its range: the
      // other piece was its CTA's first, stored long ago. One of more pieces is finished by all
      // of its CTAs, below.
      int first = 0, pieces = 1;  // of the item: CTA of the first piece, pieces
      if (!(u.begins && u.ends)) {
        const int g0 = plan.range_of(u.item_end - (ceil_div(u.ctx, kNK) + u.nns));  // the first stage's range
        first = g0 * plan.gang + member;
        pieces = plan.range_of(u.item_end - 1) - g0 + 1;
      }
      const bool takes = pieces == 2 && u.begins, gives = pieces > 1 && !takes;
      constexpr int kChunks = D / 16 / kStreams;  // a stream's share of the output, in 16 columns
      float m2 = -INFINITY, l2 = 0.f;
      if (takes) {
        const int64_t rest = 2 * ((int64_t)blockIdx.x + plan.gang);
        if (lane == 0) {
          while (ok && ld_acquire_gpu(&p.counts[2 * first]) < 1) ok = global_ns() <= deadline;
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        m2 = ld_cg(&p.part_ml[rest * 256 + r]);
        l2 = ld_cg(&p.part_ml[rest * 256 + 128 + r]);
      }
      // The piece's streams joined: maxima and sums through shared memory, then each stream's
      // warps take their share of the output columns from every accumulator.
      if (i0 < u.nst) confirm(gs + (u.nst - 1 - i0) / kStreams * kStreams + i0);
      float* ml = s_ml + (k & 1) * kStreams * 256;
      ml[stream * 256 + r] = m;
      ml[stream * 256 + 128 + r] = l;
      tc_fence_before_sync();
      named_barrier_sync(1, SW * 32);
      if (tid == 0) {
        mbar_arrive(&q_free[k & 1]);  // every stream's last O is done, so every S is
        if (takes) st_relaxed_gpu(&p.counts[2 * first], 0);  // as the next call needs it
      }
      tc_fence_after_sync();
      if (!ok) report(p.status, PKV_ERR_TIMEOUT);
      if (live) {
        float top = -INFINITY, sum = 0.f, wgt[kStreams];
#pragma unroll
        for (int s = 0; s < kStreams; ++s) top = fmaxf(top, ml[s * 256 + r]);
        const float mref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int s = 0; s < kStreams; ++s) {
          wgt[s] = ex2(ml[s * 256 + r] - mref);
          sum += wgt[s] * ml[s * 256 + 128 + r];
        }
        const int64_t slot = 2 * (int64_t)blockIdx.x + u.begins;
        float w_rest = 0.f;
        if (takes) {
          const float all = fmaxf(top, m2), aref = all == -INFINITY ? 0.f : all, w_own = ex2(top - aref);
          w_rest = ex2(m2 - aref);
          sum = w_own * sum + w_rest * l2;
#pragma unroll
          for (int s = 0; s < kStreams; ++s) wgt[s] *= w_own;
        }
        if (gives && stream == 0) {
          p.part_ml[slot * 256 + r] = top;
          p.part_ml[slot * 256 + 128 + r] = sum;
        }
        const float inv = gives ? 1.f : sum > 0.f || sum != sum ? 1.f / sum : 0.f;  // no visible key: zeros
        T* orow = reinterpret_cast<T*>(p.out) + node * p.out_st + (int64_t)(u.head * G + gq) * p.out_sh;
#pragma unroll
        for (int share = 0; share < kChunks; ++share) {
          const int c = stream + share * kStreams;
          float acc[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] = 0.f;
          if (takes) {
            const float4* const rest = p.part_o + (2 * ((int64_t)blockIdx.x + plan.gang) * (D / 4) + c * 4) * 128 + r;
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 v = ld_cg(rest + e / 4 * 128);
              acc[e] = w_rest * v.x, acc[e + 1] = w_rest * v.y, acc[e + 2] = w_rest * v.z, acc[e + 3] = w_rest * v.w;
            }
          }
#pragma unroll
          for (int s = 0; s < kStreams; ++s) {
            if (first_of(s, gs) >= u.nst) continue;  // its accumulator holds nothing of this piece
            uint32_t ob[16];
            tmem_ld16(tl + S::OCOL + s * D + c * 16, ob);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] += wgt[s] * __uint_as_float(ob[e]);
          }
          if (!valid || !ok) continue;
          if (gives) {
            float4* po = p.part_o + (slot * (D / 4) + c * 4) * 128 + r;
#pragma unroll
            for (int e = 0; e < 16; e += 4) po[e / 4 * 128] = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
          } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = Dt<T>::pack(acc[2 * e] * inv, acc[2 * e + 1] * inv);
            if (p.out_vec16) {
              *reinterpret_cast<uint4*>(orow + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(orow + c * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) reinterpret_cast<uint32_t*>(orow + c * 16)[e] = w[e];
            }
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int x = 0; x < kStreams; ++x)
          if (first_of(x, gs) < u.nst) mbar_arrive(&o_free[x]);
      }
      if (gives) {  // the piece's state is stored: count it
        named_barrier_sync(1, SW * 32);
        if (tid == 0) {
          if (pieces > 2)
            s_cut[u.begins] = CutPiece{(int)node, u.head, u.rows, pieces, range - quotient(first, plan.gang), first};
          atom_add_acq_rel_gpu(&p.counts[2 * first], 1);
        }
      }
    }
    // ---------------------------------------------------------------- join of items of three pieces and more
    // With M the largest of an item's pieces' maxima,
    //   out = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.
    // The item's CTAs each wait for all of its pieces (a CTA has stored its own two before it
    // waits for anyone's, and all CTAs are resident) and take a share of the columns, so an
    // item cut into many pieces has as many CTAs to read them. The pieces' maxima go to
    // shared memory, over the drained rings; a thread takes one row.
    named_barrier_sync(1, SW * 32);
    deadline = global_ns() + kWaitBudgetNs;
    if (tid == 0 || tid == 32) {  // a range has at most two such pieces: one thread waits for each
      const int side = tid / 32;
      const CutPiece cut = s_cut[side];
      if (cut.pieces > 0) {
        int32_t* const counts = p.counts + 2 * cut.first;
        bool all = true;
        while (all && ld_acquire_gpu(counts) < cut.pieces) all = global_ns() <= deadline;
        if (!all) report(p.status, PKV_ERR_TIMEOUT);
        // Whoever is last to see the count complete leaves the counters as the next call needs them.
        if (all && atomicAdd(counts + 1, 1) == cut.pieces - 1) {
          st_relaxed_gpu(counts, 0);
          st_relaxed_gpu(counts + 1, 0);
        }
        s_joins[side] = all;
      }
    }
    named_barrier_sync(1, SW * 32);
    for (int side = 0; side < 2; ++side) {
      const CutPiece cut = s_cut[side];
      if (cut.pieces == 0 || !s_joins[side]) continue;
      // Quads of columns: this CTA's share, the streams' warps taking every other one; about
      // D / 8 quads of states per thread however many pieces there are. Loads (past L1, which
      // other CTAs' stores do not reach) go out sixteen at a time, quad by quad and piece by
      // piece, the first of them before the weights are known.
      const bool joins = r < cut.rows;
      const int last = cut.pieces - 1, q0 = cut.index * (D / 4) / cut.pieces + stream;
      const int q_end = (cut.index + 1) * (D / 4) / cut.pieces;
      auto slot_of = [&](int x) { return 2 * ((int64_t)cut.first + x * plan.gang) + (x == 0); };
      float4 v[16];
      int fx = 0, fq = q0;  // piece and quad of the next load
      auto fetch = [&]() {
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          v[y] = ld_cg(p.part_o + (slot_of(fx) * (D / 4) + min(fq, D / 4 - 1)) * 128 + r);
          if (fx == last) fx = 0, fq += kStreams;
          else ++fx;
        }
      };
      if (joins && q0 < q_end) fetch();
      // Each stream's warps read every other piece's maximum and sum.
      float* const maxima = reinterpret_cast<float*>(smem) + side * s_cut[0].pieces * 128 + r;  // [pieces] of this row
      float* const ml = s_ml + side * kStreams * 256 + r;
      float top = -INFINITY, sum = 0.f;
      if (joins) {
        for (int x0 = stream; x0 <= last; x0 += 8 * kStreams) {
          float m8[8], l8[8], most = top, part = 0.f;
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const int64_t at = slot_of(min(x0 + y * kStreams, last)) * 256 + r;
            m8[y] = ld_cg(&p.part_ml[at]);
            l8[y] = ld_cg(&p.part_ml[at + 128]);
          }
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            if (x0 + y * kStreams > last) continue;
            maxima[(x0 + y * kStreams) * 128] = m8[y];
            most = fmaxf(most, m8[y]);
          }
          const float mref = most == -INFINITY ? 0.f : most;
#pragma unroll
          for (int y = 0; y < 8; ++y)
            if (x0 + y * kStreams <= last) part += ex2(m8[y] - mref) * l8[y];
          sum = sum * ex2(top - mref) + part;
          top = most;
        }
      }
      ml[stream * 256] = top;
      ml[stream * 256 + 128] = sum;
      named_barrier_sync(1, SW * 32);
      if (joins) {
        const float t2 = ml[(1 - stream) * 256], all = fmaxf(top, t2), mref = all == -INFINITY ? 0.f : all;
        sum = sum * ex2(top - mref) + ml[(1 - stream) * 256 + 128] * ex2(t2 - mref);
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        T* orow = reinterpret_cast<T*>(p.out) + ((int64_t)cut.node + t) * p.out_st + (int64_t)(cut.head * G + gq) * p.out_sh;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        int x = 0, q = q0;
        while (q < q_end) {
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            if (q >= q_end) continue;
            const float w = ex2(maxima[x * 128] - mref);
            acc.x += w * v[y].x, acc.y += w * v[y].y, acc.z += w * v[y].z, acc.w += w * v[y].w;
            if (x++ < last) continue;
            uint32_t* o = reinterpret_cast<uint32_t*>(orow + 4 * q);
            o[0] = Dt<T>::pack(acc.x * inv, acc.y * inv);
            o[1] = Dt<T>::pack(acc.z * inv, acc.w * inv);
            acc = make_float4(0.f, 0.f, 0.f, 0.f);
            x = 0;
            q += kStreams;
          }
          if (q < q_end) fetch();
        }
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    if (!mbar_wait_until(mma_done, 0, global_ns() + kWaitBudgetNs) && lane == 0) report(p.status, PKV_ERR_TIMEOUT);
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::NCOLS);
  }
}

int tree_ctas() { return std::min(num_sms(), kMaxPieces); }
constexpr int kCountBytes = 4096;  // the items' counters, at the front of the workspace

template <typename T, int D>
int launch(const CUtensorMap (&maps)[5], const TreeParams& p, cudaStream_t st) {
  using S = TreeShape<D>;
  static SmemAttribute attribute;
  const cudaError_t e = attribute.set(reinterpret_cast<const void*>(tree_kernel<T, D>), S::SMEM);
  if (e != cudaSuccess) return cuda_status(e);
  // Cooperative: the CTAs wait for one another's pieces, so they must all be resident.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tree_ctas());
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, tree_kernel<T, D>, maps[0], maps[1], maps[2], maps[3], maps[4], p));
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_tree_attention_workspace_bytes(int32_t batch, int32_t head_dim) {
  if (batch <= 0 || batch > kMaxSeqs || (head_dim != 64 && head_dim != 128)) return 0;
  return kCountBytes + 2 * (int64_t)tree_ctas() * 128 * (head_dim + 2) * 4;
}

extern "C" int pkv_tree_attention(const pkv_pool* pool, int32_t layer, const pkv_tables* tables, int32_t num_seqs,
                                  const int32_t* cu_nodes, const int32_t* context_lens, int32_t max_nodes,
                                  int64_t total_nodes, int32_t num_q_heads, void* out, int64_t out_stride_n,
                                  int64_t out_stride_h, const void* q, int64_t q_stride_n, int64_t q_stride_h,
                                  const void* k_nodes, int64_t k_stride_n, int64_t k_stride_h, const void* v_nodes,
                                  int64_t v_stride_n, int64_t v_stride_h, const int64_t* mask, int32_t mask_words,
                                  float scale, void* workspace, int64_t workspace_bytes, int32_t* status_dev,
                                  pkv_stream_t stream) {
  if (!pool || !pool->k || !pool->v || !tables) return PKV_ERR_INVALID_ARGUMENT;
  if (num_seqs < 0 || max_nodes < 0 || total_nodes < 0 || total_nodes > 0x7fffffff - 4096 || layer < 0 ||
      layer >= pool->num_layers || pool->num_blocks_total <= 0 || mask_words <= 0 || !(scale > 0.f) || num_q_heads <= 0 ||
      pool->num_kv_heads <= 0 || num_q_heads % pool->num_kv_heads || tables->cols <= 0 || tables->rows <= 0 ||
      tables->stride < 0 || (!tables->seq_rows && tables->rows < num_seqs) || tables->cols > (1 << 26))
    return PKV_ERR_INVALID_ARGUMENT;
  const int d = pool->head_dim, hkv = pool->num_kv_heads, group = num_q_heads / hkv;
  if (pool->block_size != kBS || (d != 64 && d != 128) || group > 16 || num_seqs > kMaxSeqs || hkv > 1024 ||
      mask_words > kMaxWords || (pool->dtype != PKV_F16 && pool->dtype != PKV_BF16))
    return PKV_ERR_UNSUPPORTED;
  if (max_nodes > 64 * mask_words) return PKV_ERR_INVALID_ARGUMENT;
  // Stages are counted in 32 bits: every tile of every head against a full table row.
  const int64_t tiles = std::min((int64_t)num_seqs * ((max_nodes + 128 / group - 1) / (128 / group)),
                                 total_nodes / (128 / group) + num_seqs);
  if (tiles * hkv * (kItemCost + 2 + max_nodes / kNK + tables->cols / (kNK / kBS)) > 0x7fffffff) return PKV_ERR_UNSUPPORTED;
  if (num_seqs == 0 || total_nodes == 0) return PKV_OK;
  if (!tables->block_tables || !cu_nodes || !context_lens || !out || !q || !k_nodes || !v_nodes || !mask)
    return PKV_ERR_INVALID_ARGUMENT;
  auto addr = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
  if ((addr(out) & 3) || ((out_stride_n | out_stride_h) & 1)) return PKV_ERR_INVALID_ARGUMENT;
  // Q and the nodes' K/V are read by TMA: rows and heads on 16 bytes.
  const int64_t strides[6] = {q_stride_n, q_stride_h, k_stride_n, k_stride_h, v_stride_n, v_stride_h};
  const int64_t steps[6] = {total_nodes, num_q_heads, total_nodes, hkv, total_nodes, hkv};
  if ((addr(q) | addr(k_nodes) | addr(v_nodes)) & 15) return PKV_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 6; ++i)
    if (strides[i] < (steps[i] > 1) || strides[i] % 8 || strides[i] >= (int64_t)1 << 38) return PKV_ERR_INVALID_ARGUMENT;
  if (!workspace || (addr(workspace) & 255)) return PKV_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < pkv_tree_attention_workspace_bytes(num_seqs, d)) return PKV_ERR_WORKSPACE;
  CUtensorMap maps[5];
  if (!get_pool_maps(*pool, &maps[0], &maps[1], kRowGroups)) return PKV_ERR_CUDA;
  int rc = make_row_group_tensor_map(&maps[2], k_nodes, pool->dtype, d, hkv, total_nodes, k_stride_h, k_stride_n);
  if (rc == PKV_OK)
    rc = make_row_group_tensor_map(&maps[3], v_nodes, pool->dtype, d, hkv, total_nodes, v_stride_h, v_stride_n);
  if (rc == PKV_OK)
    rc = make_rows_tensor_map(&maps[4], q, pool->dtype, d, num_q_heads, total_nodes, q_stride_h, q_stride_n, group,
                              128 / group);
  if (rc != PKV_OK) return rc;
  TreeParams p;
  p.out = out;
  p.cu = cu_nodes;
  p.ctx = context_lens;
  p.mask = reinterpret_cast<const uint64_t*>(mask);
  p.tables = tables->block_tables;
  p.seq_rows = tables->seq_rows;
  p.status = status_dev;
  p.counts = static_cast<int32_t*>(workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCountBytes);
  p.part_o = reinterpret_cast<float4*>(p.part_ml + 2 * (int64_t)tree_ctas() * 256);
  p.out_st = out_stride_n, p.out_sh = out_stride_h;
  p.table_stride = tables->stride;
  p.total_nodes = total_nodes;
  p.table_rows = tables->rows;
  p.table_cols = tables->cols;
  p.batch = num_seqs;
  p.hkv = hkv;
  p.group = group;
  p.tile_nodes = 128 / group;
  p.words = mask_words;
  p.layer = layer;
  p.nbt = pool->num_blocks_total;
  p.max_nodes = max_nodes;
  p.scale_log2 = scale * kLog2e;
  p.out_vec16 = (addr(out) & 15) == 0 && ((out_stride_n | out_stride_h) & 7) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pool->dtype == PKV_F16)
    return d == 64 ? launch<__half, 64>(maps, p, st) : launch<__half, 128>(maps, p, st);
  return d == 64 ? launch<__nv_bfloat16, 64>(maps, p, st) : launch<__nv_bfloat16, 128>(maps, p, st);
}
