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
// Work split. Unit = (sequence, run of context stages of 64 keys, KV head, tile of 128
// rows); the first run also takes the tree's own keys. Every CTA derives the same split
// from the lengths on the device: its ten warps try run lengths of 2 .. 128 stages (and
// whole contexts) and the one with the least cost, waves x (run + overhead), wins; nothing
// of the plan needs the host to know a length. A sequence left whole writes its output; one
// cut into several runs leaves per-run states (running maximum, sum, unnormalised output,
// all float32) that a second small kernel joins. Tiles of one run come next to each other,
// so that a wide tree's tiles read the same keys from L2 at the same time.
//
// Inside a CTA: one warp issues the TMA copies (K and V rings of their own), one thread the
// tcgen05 MMAs, the others the softmax. S = Q K^T (128 x 64, float32 in TMEM, Q resident in
// TMEM), P = 2^(S - m) rounded to the storage type over S in its own buffer (two buffers in
// turn), O += P V in TMEM against a maximum m that moves only when a row's maximum grew by
// more than 8 (in log2). Rounding P costs each weight half a step of its type, as much as
// the output's own rounding; the row sum is taken before it, in float32.
#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"

namespace pkv {
namespace {

constexpr int kBS = 16;
constexpr int kNK = 64;          // keys per stage
constexpr int kKS = 4;           // K ring stages
constexpr int kVS = 4;           // V ring stages
constexpr int kBars = 2 * (kKS + kVS) + 4;
constexpr int kMaxSeqs = 1024;   // sequences per call: their tables live in shared memory
constexpr int kMaxWords = 8;     // mask words of 64 nodes
constexpr int kWaves = 2;        // cut units per resident CTA that the workspace has room for
constexpr float kLog2e = 1.4426950408889634f;
// Run lengths (stages) the plan tries; the last leaves every context whole.
constexpr int kRuns = 20;
__host__ __device__ constexpr int run_candidate(int i) {
  constexpr int runs[kRuns] = {2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32, 40, 48, 64, 96, 128, 1 << 24};
  return runs[i];
}
constexpr int kUnitCost = 4;     // a unit's start and end, in stages
constexpr int kJoinCost = 4;     // the join and its traffic, in stages

template <int D> struct TreeShape {
  static constexpr int DC = D / 64;             // 64-wide head_dim chunks
  static constexpr int KSB = DC * kNK * 128;    // one stage of K (or V): [DC][64 keys][64], 128B-swizzled
  // TMEM columns: two S / P buffers, O, Q (packed 16-bit pairs).
  static constexpr int OCOL = 2 * kNK;
  static constexpr int QCOL = OCOL + D;
  static constexpr int NCOLS = QCOL + D / 2 <= 256 ? 256 : 512;
  static constexpr int MIN_BLOCKS = NCOLS <= 256 ? 2 : 1;
  static constexpr int SW = MIN_BLOCKS == 2 ? 4 : 8;  // softmax warps: a row, or half a row, per thread
  static constexpr int HALVES = SW / 4;
  static constexpr int THREADS = (SW + 2) * 32;
  static constexpr int SMEM = 1024 + (kKS + kVS) * KSB + (kBars + 2) * 8 + 3 * 2 * 128 * 4 + (3 * kMaxSeqs + 2) * 4;
};

struct TreeParams {
  void* out;
  const void* q;
  const int32_t* cu;
  const int32_t* ctx;
  const uint64_t* mask;
  const int32_t* tables;
  const int32_t* seq_rows;
  int32_t* status;
  int32_t* plan;       // [0] run length, [1 + b] first unit of sequence b
  float* part_ml;      // [units][2][128] running maximum and sum
  float* part_o;       // [units][D][128]
  int64_t out_st, out_sh, q_st, q_sh, table_stride, total_nodes;
  int32_t table_rows, table_cols, batch, hkv, group, tile_nodes, words, layer, nbt, max_units;
  int32_t q_vec16, out_vec16, max_nodes;
  float scale_log2;
};

__device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Tiles, context stages and runs of a sequence with n nodes and c cached keys.
__device__ inline int runs_of(int stages, int run) { return max(1, ceil_div(stages, run)); }

// 4-D bulk tensor copy global -> shared (no multicast), completion on an mbarrier.
__device__ inline void tma_load_4d(void* smem_dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                   uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(TreeShape<D>::THREADS, TreeShape<D>::MIN_BLOCKS)
    tree_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                const __grid_constant__ CUtensorMap nmap_k, const __grid_constant__ CUtensorMap nmap_v,
                const TreeParams p) {
  using S = TreeShape<D>;
  constexpr int DC = S::DC, SW = S::SW, HALVES = S::HALVES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;                     // [kKS][KSB]
  uint8_t* sV = sK + kKS * S::KSB;        // [kVS][KSB]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kVS * S::KSB);
  uint64_t* k_full = bars;                // [kKS] K landed
  uint64_t* v_full = k_full + kKS;        // [kVS] V landed
  uint64_t* s_done = v_full + kVS;        // [kKS] S(j) = Q K(j)^T done: S ready, K stage free
  uint64_t* o_done = s_done + kKS;        // [kVS] O += P(j) V(j) done: V stage free
  uint64_t* p_full = o_done + kVS;        // [2] P(j) stored, j even / odd
  uint64_t* q_ready = p_full + 2;         // Q stored
  uint64_t* mma_done = q_ready + 1;       // every MMA of the CTA completed
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + kBars);
  float* s_mx = reinterpret_cast<float*>(bars + kBars + 2);  // [2 parities][2 halves][128] partial maxima
  float* s_l = s_mx + 2 * 2 * 128;                           // [2 halves][128] partial sums
  int32_t* s_cu = reinterpret_cast<int32_t*>(s_l + 2 * 128);  // [batch + 1]
  int32_t* s_ctx = s_cu + kMaxSeqs + 1;                       // [batch] cached keys
  int32_t* s_unit = s_ctx + kMaxSeqs;                         // [batch + 1] units before sequence b
  __shared__ uint64_t s_cost[kRuns];
  __shared__ int s_warp[16], s_stages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = p.batch, G = p.group;

  grid_dep_launch_dependents();  // the join's CTAs may wait in place
  if (tid == 0) {
    for (int i = 0; i < kKS; ++i) mbar_init(&k_full[i], 1), mbar_init(&s_done[i], 1);
    for (int i = 0; i < kVS; ++i) mbar_init(&v_full[i], 1), mbar_init(&o_done[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&p_full[i], SW);
    mbar_init(q_ready, SW);
    mbar_init(mma_done, 1);
    fence_mbar_init();
    s_stages = 0;
  }
  if (warp == 0) {
    tmem_alloc(tslot, S::NCOLS);
    tc_fence_before_sync();
  }
  if (warp == SW && lane == 0) {
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
    prefetch_tensormap(&nmap_k);
    prefetch_tensormap(&nmap_v);
  }
  // ------------------------------------------------------------------ plan
  // Lengths, clamped to what the call's own sizes allow (a bad one is reported and its
  // sequence shortened, so every index below stays in range).
  for (int b = tid; b <= B; b += S::THREADS) {
    int c = p.cu[b];
    if (c < 0 || c > p.total_nodes) {
      report(p.status, PKV_ERR_OUT_OF_RANGE);
      c = (int)min((int64_t)max(c, 0), p.total_nodes);
    }
    s_cu[b] = c;
    if (b < B) {
      int n = p.ctx[b];
      if (n < 0 || n > (int64_t)p.table_cols * kBS) {
        report(p.status, PKV_ERR_OUT_OF_RANGE);
        n = (int)min((int64_t)max(n, 0), (int64_t)p.table_cols * kBS);
      }
      const int row = p.seq_rows ? p.seq_rows[b] : b;
      if (row >= p.table_rows) report(p.status, PKV_ERR_OUT_OF_RANGE);
      if (row < 0 || row >= p.table_rows) n = 0;  // a padding row has no cached keys
      s_ctx[b] = n;
    }
  }
  __syncthreads();
  auto nodes_of = [&](int b) {
    const int n = s_cu[b + 1] - s_cu[b];
    return n < 0 ? 0 : min(n, p.max_nodes);
  };
  {
    int most = 0;
    for (int b = tid; b < B; b += S::THREADS) {
      const int n = s_cu[b + 1] - s_cu[b];
      if (n < 0 || n > p.max_nodes) report(p.status, PKV_ERR_OUT_OF_RANGE);
      most = max(most, ceil_div(s_ctx[b], kNK));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&s_stages, most);
  }
  __syncthreads();
  const int max_stages = s_stages;
  for (int c = warp; c < kRuns; c += SW + 2) {
    const int run = run_candidate(c);
    int64_t units = 0;
    for (int b = lane; b < B; b += 32)
      units += (int64_t)ceil_div(nodes_of(b), p.tile_nodes) * p.hkv * runs_of(ceil_div(s_ctx[b], kNK), run);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
    if (lane == 0) {
      const bool cut = run < max_stages;
      const int64_t waves = (units + gridDim.x - 1) / gridDim.x;
      s_cost[c] = cut && units > p.max_units ? ~0ull  // more states than the workspace holds
                                             : waves * (min(run, max_stages) + kUnitCost) + (cut ? kJoinCost : 0);
    }
  }
  __syncthreads();
  int best = 0;
#pragma unroll
  for (int c = 1; c < kRuns; ++c)
    if (s_cost[c] < s_cost[best]) best = c;
  const int run = run_candidate(best);
  // Units before each sequence: a scan over the CTA, a few sequences per thread.
  {
    const int per = ceil_div(B, S::THREADS), b0 = min(B, tid * per), b1 = min(B, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; ++b)
      mine += ceil_div(nodes_of(b), p.tile_nodes) * p.hkv * runs_of(ceil_div(s_ctx[b], kNK), run);
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int before = inc - mine;
    for (int w = 0; w < warp; ++w) before += s_warp[w];
    for (int b = b0; b < b1; ++b) {
      s_unit[b] = before;
      if (blockIdx.x == 0) p.plan[1 + b] = before;
      before += ceil_div(nodes_of(b), p.tile_nodes) * p.hkv * runs_of(ceil_div(s_ctx[b], kNK), run);
    }
    if (b1 == B && b0 < B) s_unit[B] = before;
    if (blockIdx.x == 0 && tid == 0) p.plan[0] = run;
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tslot;
  const uint64_t deadline = global_ns() + kWaitBudgetNs;
  auto s_col = [](int b) { return (uint32_t)(b * kNK); };
  const int n_units = s_unit[B];

  // Every role walks the same units and numbers stages across them, so ring slots and
  // barrier parities continue from one unit to the next.
  struct Unit {
    int b, head, tile, rows, n, ctx, first, nst, nns;  // nns: leading stages of the tree's own keys
    bool cut;
  };
  auto unit_at = [&](int w) {
    Unit u;
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_unit[mid] <= w) lo = mid; else hi = mid - 1;
    }
    u.b = lo;
    u.n = nodes_of(lo);
    u.ctx = s_ctx[lo];
    const int tiles = ceil_div(u.n, p.tile_nodes), cst = ceil_div(u.ctx, kNK), ch = runs_of(cst, run);
    int r = w - s_unit[lo];
    u.tile = r % tiles;
    r /= tiles;
    u.head = r % p.hkv;
    const int k = r / p.hkv;
    u.rows = min(p.tile_nodes, u.n - u.tile * p.tile_nodes) * G;
    u.first = (int)((int64_t)k * cst / ch);
    u.nns = k == 0 ? ceil_div(u.n, kNK) : 0;
    u.nst = u.nns + (int)((int64_t)(k + 1) * cst / ch) - u.first;
    u.cut = ch > 1;
    return u;
  };

  if (warp == SW) {
    // ---------------------------------------------------------------- TMA copies
    constexpr int kCopies = (kNK / kBS) * DC;  // a context stage: one copy per lane
    const int bl = lane / DC, c = lane % DC;
    bool ok = true;
    int gs = 0;
    for (int w = blockIdx.x; w < n_units && ok; w += gridDim.x) {
      const Unit u = unit_at(w);
      int row = p.seq_rows ? p.seq_rows[u.b] : u.b;
      const int32_t* table = row >= 0 && row < p.table_rows ? p.tables + (int64_t)row * p.table_stride : nullptr;
      const int nkb = ceil_div(u.ctx, kBS), kb0 = u.first * (kNK / kBS);
      auto lookup = [&](int kb) -> int {  // blocks past the sequence: masked, any block will do
        int blk = kb < nkb && table ? table[kb] : p.nbt - 1;
        if (blk < 0 || blk >= p.nbt) {
          report(p.status, PKV_ERR_OUT_OF_RANGE);
          blk = p.nbt - 1;
        }
        return blk;
      };
      constexpr int kPerWindow = 32 / (kNK / kBS);  // stages per window of 32 block ids
      int win = lookup(kb0 + lane), win_next = lookup(kb0 + 32 + lane);
      for (int i = 0; i < u.nst && ok; ++i) {
        const int ci = i - u.nns;  // context stage of the unit
        int blk = 0;
        if (ci >= 0) {
          if (ci > 0 && ci % kPerWindow == 0) {
            win = win_next;
            win_next = lookup(kb0 + 32 * (ci / kPerWindow + 1) + lane);
          }
          blk = __shfl_sync(0xffffffffu, win, (ci * (kNK / kBS) + bl) % 32);
        }
        const int c4 = p.layer * p.nbt + blk, j = gs + i, sk = j % kKS, sv = j % kVS;
        const int node = s_cu[u.b] + i * kNK;
        if (lane == 0) {
          if (j >= kKS && !mbar_wait_until(&s_done[sk], ((j / kKS) - 1) & 1, deadline)) {
            report(p.status, PKV_ERR_TIMEOUT);
            ok = false;
          }
          if (ok) mbar_arrive_expect_tx(&k_full[sk], S::KSB);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (ok && ci >= 0 && lane < kCopies)
          tma_load_5d(sK + sk * S::KSB + c * kNK * 128 + bl * kBS * 128, &tmap_k, 0, 0, c, u.head, c4, &k_full[sk]);
        if (ok && ci < 0 && lane < DC) tma_load_4d(sK + sk * S::KSB + lane * kNK * 128, &nmap_k, 0, lane, u.head, node, &k_full[sk]);
        if (lane == 0 && ok) {
          if (j >= kVS && !mbar_wait_until(&o_done[sv], ((j / kVS) - 1) & 1, deadline)) {
            report(p.status, PKV_ERR_TIMEOUT);
            ok = false;
          }
          if (ok) mbar_arrive_expect_tx(&v_full[sv], S::KSB);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (ok && ci >= 0 && lane < kCopies)
          tma_load_5d(sV + sv * S::KSB + c * kNK * 128 + bl * kBS * 128, &tmap_v, 0, 0, c, u.head, c4, &v_full[sv]);
        if (ok && ci < 0 && lane < DC) tma_load_4d(sV + sv * S::KSB + lane * kNK * 128, &nmap_v, 0, lane, u.head, node, &v_full[sv]);
      }
      gs += u.nst;
    }
  } else if (warp == SW + 1) {
    // ---------------------------------------------------------------- MMA issue
    if (lane == 0) {
      constexpr bool kBf16 = Dt<T>::code == PKV_BF16;
      constexpr uint32_t idesc_s = umma_idesc_f16(kBf16, false, 128, kNK);
      constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, true, 128, D);
      auto pin = [](uint64_t& x) { asm volatile("" : "+l"(x)); };
      auto issue_s = [&](int j, bool after_o) -> bool {  // S(j) into buffer j % 2, over P(j - 2)
        const int st = j % kKS, b = j % 2;
        uint64_t bk[D / 16];
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          bk[kk] = umma_desc_sw128(smem_u32(sK + st * S::KSB + (kk / 4) * kNK * 128 + (kk % 4) * 32), 16, 1024);
          pin(bk[kk]);
        }
        if (!mbar_wait_until(&k_full[st], (j / kKS) & 1, deadline)) return false;
        if (after_o && !mbar_wait_until(&o_done[(j - 2) % kVS], ((j - 2) / kVS) & 1, deadline)) return false;
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_ts(tmem + s_col(b), tmem + S::QCOL + kk * 8, bk[kk], idesc_s, kk > 0);
        umma_commit(&s_done[st]);
        return true;
      };
      auto issue_o = [&](int j, bool first) -> bool {
        const int st = j % kVS, b = j % 2;
        uint64_t bv[kNK / 16];
#pragma unroll
        for (int kb = 0; kb < kNK / 16; ++kb) {
          bv[kb] = umma_desc_sw128(smem_u32(sV + st * S::KSB + kb * 16 * 128), kNK * 128, 1024);
          pin(bv[kb]);
        }
        if (!mbar_wait_until(&p_full[b], (j / 2) & 1, deadline)) return false;
        if (!mbar_wait_until(&v_full[st], (j / kVS) & 1, deadline)) return false;
        tc_fence_after_sync();
#pragma unroll
        for (int kb = 0; kb < kNK / 16; ++kb)
          umma_f16_ts(tmem + S::OCOL, tmem + s_col(b) + kb * 8, bv[kb], idesc_o, !first || kb > 0);
        umma_commit(&o_done[st]);
        return true;
      };
      bool ok = true;
      int gs = 0, k = 0;
      for (int w = blockIdx.x; w < n_units && ok; w += gridDim.x, ++k) {
        const int nst = unit_at(w).nst;
        ok = mbar_wait_until(q_ready, k & 1, deadline) && issue_s(gs, false) && (nst < 2 || issue_s(gs + 1, false));
        for (int i = 0; i < nst && ok; ++i) ok = issue_o(gs + i, i == 0) && (i + 2 >= nst || issue_s(gs + i + 2, true));
        gs += nst;
      }
      if (!ok) report(p.status, PKV_ERR_TIMEOUT);
      if (k > 0) umma_commit(mma_done); else mbar_arrive(mma_done);
    }
  } else {
    // ---------------------------------------------------------------- softmax warps
    constexpr int KH = kNK / HALVES, DH = D / HALVES;
    const int hf = warp / 4;
    const int r = (warp % 4) * 32 + lane;  // TMEM lane = tile row
    const int t = r / G, gq = r - t * G;   // node of the tile, query head of the group
    const uint32_t tl = tmem + ((uint32_t)((warp % 4) * 32) << 16);
    const int pair_bar = 1 + warp % 4;     // the two warps of a row
    constexpr float kSlack = 8.f;
    bool ok = true;
    auto confirm = [&](int j) {
      if (ok && !mbar_wait_until(&o_done[j % kVS], (j / kVS) & 1, deadline)) ok = false;
    };
    int gs = 0;
    for (int w = blockIdx.x; w < n_units; w += gridDim.x) {
      const Unit u = unit_at(w);
      const int nst = u.nst;
      const bool valid = r < u.rows;
      const bool live = (warp % 4) * 32 < u.rows;  // some row of the warp has a query
      const int64_t node = (int64_t)s_cu[u.b] + u.tile * p.tile_nodes + t;
      {
        const T* qrow = reinterpret_cast<const T*>(p.q) + node * p.q_st + (int64_t)(u.head * G + gq) * p.q_sh + hf * DH;
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {
          uint32_t qv[16];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (valid) {
              if (p.q_vec16) {
                v = *reinterpret_cast<const uint4*>(qrow + c * 32 + 8 * k);
              } else {
                const uint32_t* q32 = reinterpret_cast<const uint32_t*>(qrow + c * 32 + 8 * k);
                v = make_uint4(q32[0], q32[1], q32[2], q32[3]);
              }
            }
            qv[4 * k] = v.x, qv[4 * k + 1] = v.y, qv[4 * k + 2] = v.z, qv[4 * k + 3] = v.w;
          }
          tmem_st16(tl + S::QCOL + hf * (DH / 2) + c * 16, qv);
        }
      }
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);

      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < nst; ++i) {
        const int j = gs + i, b = j % 2;
        const bool own = i < u.nns;  // the tree's own keys
        const int keys = own ? u.n - i * kNK : u.ctx - (u.first + i - u.nns) * kNK;  // keys of the stage, if < kNK
        uint64_t see = ~0ull;
        if (own) see = valid ? p.mask[node * p.words + i] : 0;
        if (keys < kNK) see &= (1ull << keys) - 1;
        if (ok && !mbar_wait_until(&s_done[j % kKS], (j / kKS) & 1, deadline)) ok = false;
        tc_fence_after_sync();
        // Rows of V past the sequence or the tree hold whatever was there, infinities and NaN
        // included: 0 x NaN would reach the output, so they are cleared in place.
        if (keys < kNK) {
          const int st = j % kVS;
          if (ok && !mbar_wait_until(&v_full[st], (j / kVS) & 1, deadline)) ok = false;
          for (int x = tid; x < (kNK - keys) * DC * 8; x += SW * 32) {
            const int c = x / ((kNK - keys) * 8), y = x - c * (kNK - keys) * 8;
            *reinterpret_cast<uint4*>(sV + st * S::KSB + c * kNK * 128 + keys * 128 + y * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        if (live) {
          uint32_t sa[KH];
#pragma unroll
          for (int c = 0; c < KH / 32; ++c)
            tmem_ld32(tl + s_col(b) + hf * KH + c * 32, *reinterpret_cast<uint32_t(*)[32]>(sa + c * 32));
          tmem_wait_ld();
          if (own || keys < kNK) {
            const uint32_t lo32 = (uint32_t)(see >> (hf * KH)), hi32 = KH > 32 ? (uint32_t)(see >> 32) : 0;
#pragma unroll
            for (int e = 0; e < KH; ++e)
              if (!((e < 32 ? lo32 >> (e & 31) : hi32 >> (e & 31)) & 1)) sa[e] = __float_as_uint(-INFINITY);
          }
          float mt[KH / 2];
#pragma unroll
          for (int e = 0; e < KH / 2; ++e) mt[e] = fmaxf(__uint_as_float(sa[e]), __uint_as_float(sa[e + KH / 2]));
#pragma unroll
          for (int x = KH / 4; x > 0; x >>= 1) {
#pragma unroll
            for (int e = 0; e < x; ++e) mt[e] = fmaxf(mt[e], mt[e + x]);
          }
          float mx = mt[0] * p.scale_log2;
          if (HALVES == 2) {
            float* mxb = s_mx + (j % 2) * 256;
            mxb[hf * 128 + r] = mx;
            named_barrier_sync(pair_bar, 64);
            mx = fmaxf(mx, mxb[(1 - hf) * 128 + r]);
          }
          const float m_cand = fmaxf(m, mx);
          float alpha = 1.f;
          if (m_cand - m > kSlack) {
            alpha = ex2(m - m_cand);
            m = m_cand;
            l *= alpha;
          }
          if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            confirm(j - 1);
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < DH / 32; ++c) {
              uint32_t ob[32];
              tmem_ld32(tl + S::OCOL + hf * DH + c * 32, ob);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) ob[e] = __float_as_uint(__uint_as_float(ob[e]) * alpha);
              tmem_st32(tl + S::OCOL + hf * DH + c * 32, ob);
            }
          }
          const float mref = m == -INFINITY ? 0.f : m;
          float2 lsum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), negm2 = make_float2(-mref, -mref);
          uint32_t pk[KH / 2];
#pragma unroll
          for (int e = 0; e < KH; e += 2) {
            const float2 x = ffma2(make_float2(__uint_as_float(sa[e]), __uint_as_float(sa[e + 1])), scale2, negm2);
            const float p0 = ex2(x.x), p1 = ex2(x.y);
            pk[e / 2] = Dt<T>::pack(p0, p1);
            lsum[(e / 2) % 2] = fadd2(lsum[(e / 2) % 2], make_float2(p0, p1));
          }
          tc_fence_after_sync();
#pragma unroll
          for (int c = 0; c < KH / 32; ++c)
            tmem_st16(tl + s_col(b) + hf * (KH / 2) + c * 16, *reinterpret_cast<const uint32_t(*)[16]>(pk + c * 16));
          tmem_wait_st();
          l += (lsum[0].x + lsum[1].x) + (lsum[0].y + lsum[1].y);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
      }
      confirm(gs + nst - 1);
      tc_fence_after_sync();
      if (!ok) report(p.status, PKV_ERR_TIMEOUT);
      if (live) {
        if (HALVES == 2) {
          s_l[hf * 128 + r] = l;
          named_barrier_sync(pair_bar, 64);
          l += s_l[(1 - hf) * 128 + r];
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // no visible key: zeros
        T* orow = reinterpret_cast<T*>(p.out) + node * p.out_st + (int64_t)(u.head * G + gq) * p.out_sh + hf * DH;
        if (u.cut && hf == 0 && ok) {
          p.part_ml[(int64_t)w * 256 + r] = m;
          p.part_ml[(int64_t)w * 256 + 128 + r] = l;
        }
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {
          uint32_t ob[32];
          tmem_ld32(tl + S::OCOL + hf * DH + c * 32, ob);
          tmem_wait_ld();
          if (u.cut) {
            if (valid && ok) {
              float* po = p.part_o + ((int64_t)w * D + hf * DH + c * 32) * 128 + r;
#pragma unroll
              for (int e = 0; e < 32; ++e) po[e * 128] = __uint_as_float(ob[e]);
            }
          } else if (valid && ok) {
            auto pack = [&](int e) {
              return Dt<T>::pack(__uint_as_float(ob[e]) * inv, __uint_as_float(ob[e + 1]) * inv);
            };
            if (p.out_vec16) {
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                *reinterpret_cast<uint4*>(orow + c * 32 + e) = make_uint4(pack(e), pack(e + 2), pack(e + 4), pack(e + 6));
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 2) *reinterpret_cast<uint32_t*>(orow + c * 32 + e) = pack(e);
            }
          }
        }
      }
      gs += nst;
    }
  }
  __syncthreads();
  if (warp == 0) {
    if (!mbar_wait_until(mma_done, 0, global_ns() + kWaitBudgetNs) && lane == 0) report(p.status, PKV_ERR_TIMEOUT);
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::NCOLS);
  }
}

// Joins the runs of a cut sequence: with M the largest of their maxima,
//   out = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.
// One CTA per (8 output columns x 8, tile, KV head, sequence); a thread takes one row and
// eight columns, so the states are read a row to a lane, and its output is one 16-byte write.
constexpr int kJoinCols = 64;  // columns of a CTA: 8 threads' eight

template <typename T, int D>
__global__ void __launch_bounds__(128 * (kJoinCols / 8)) tree_join_kernel(const TreeParams p) {
  grid_dep_wait();
  const int run = p.plan[0];
  const int b = blockIdx.z, head = blockIdx.y;
  const int tile = blockIdx.x / (D / kJoinCols), part = blockIdx.x % (D / kJoinCols);
  int ctx = p.ctx[b];
  ctx = min(max(ctx, 0), p.table_cols * kBS);
  const int row = p.seq_rows ? p.seq_rows[b] : b;
  if (row < 0 || row >= p.table_rows) ctx = 0;
  const int ch = runs_of(ceil_div(ctx, kNK), run);
  if (ch == 1) return;
  const int64_t total = p.total_nodes;
  const int lo = (int)min(max((int64_t)p.cu[b], (int64_t)0), total);
  const int hi = (int)min(max((int64_t)p.cu[b + 1], (int64_t)0), total);
  const int n = hi < lo ? 0 : min(hi - lo, p.max_nodes);
  const int tiles = ceil_div(n, p.tile_nodes);
  const int r = threadIdx.x % 128, c0 = part * kJoinCols + (threadIdx.x / 128) * 8;
  if (tile >= tiles || r >= min(p.tile_nodes, n - tile * p.tile_nodes) * p.group) return;
  const int64_t step = (int64_t)p.hkv * tiles;
  const int64_t u0 = p.plan[1 + b] + (int64_t)head * tiles + tile;
  float top = -INFINITY;
  for (int k = 0; k < ch; ++k) top = fmaxf(top, p.part_ml[(u0 + k * step) * 256 + r]);
  const float mref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc[8] = {};
#pragma unroll 2
  for (int k = 0; k < ch; ++k) {
    const int64_t u = u0 + k * step;
    const float wgt = ex2(p.part_ml[u * 256 + r] - mref);
    sum += wgt * p.part_ml[u * 256 + 128 + r];
    const float* o = p.part_o + (u * D + c0) * 128 + r;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += wgt * o[e * 128];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int t = r / p.group, gq = r - t * p.group;
  T* orow = reinterpret_cast<T*>(p.out) + ((int64_t)lo + tile * p.tile_nodes + t) * p.out_st +
            (int64_t)(head * p.group + gq) * p.out_sh + c0;
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = Dt<T>::pack(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  if (p.out_vec16) {
    *reinterpret_cast<uint4*>(orow) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) reinterpret_cast<uint32_t*>(orow)[e] = w[e];
  }
}

int64_t plan_bytes(int batch) { return ((int64_t)(batch + 1) * 4 + 255) / 256 * 256; }
int resident(int d) { return num_sms() * (d == 64 ? TreeShape<64>::MIN_BLOCKS : TreeShape<128>::MIN_BLOCKS); }

template <typename T, int D>
int launch(const CUtensorMap (&maps)[4], const TreeParams& p, cudaStream_t st) {
  using S = TreeShape<D>;
  static SmemAttribute attribute;
  const cudaError_t e = attribute.set(reinterpret_cast<const void*>(tree_kernel<T, D>), S::SMEM);
  if (e != cudaSuccess) return cuda_status(e);
  tree_kernel<T, D><<<resident(D), S::THREADS, S::SMEM, st>>>(maps[0], maps[1], maps[2], maps[3], p);
  const int rc = launch_status();
  if (rc != PKV_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.max_nodes + p.tile_nodes - 1) / p.tile_nodes * (D / kJoinCols), p.hkv, p.batch);
  cfg.blockDim = dim3(128 * (kJoinCols / 8));
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, tree_join_kernel<T, D>, p));
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_tree_attention_workspace_bytes(int32_t batch, int32_t head_dim) {
  if (batch <= 0 || batch > kMaxSeqs || (head_dim != 64 && head_dim != 128)) return 0;
  return plan_bytes(batch) + (int64_t)kWaves * resident(head_dim) * 128 * (head_dim + 2) * 4;
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
  if (num_seqs == 0 || max_nodes == 0 || total_nodes == 0) return PKV_OK;
  if (!tables->block_tables || !cu_nodes || !context_lens || !out || !q || !k_nodes || !v_nodes || !mask)
    return PKV_ERR_INVALID_ARGUMENT;
  auto addr = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
  if (((addr(q) | addr(out)) & 3) || ((q_stride_n | q_stride_h | out_stride_n | out_stride_h) & 1))
    return PKV_ERR_INVALID_ARGUMENT;
  // The nodes' K/V are read by TMA: rows and heads on 16 bytes.
  if (((addr(k_nodes) | addr(v_nodes)) & 15) || ((k_stride_n | k_stride_h | v_stride_n | v_stride_h) & 7) ||
      k_stride_n < 0 || v_stride_n < 0 || k_stride_h < 0 || v_stride_h < 0)
    return PKV_ERR_INVALID_ARGUMENT;
  if (!workspace || (addr(workspace) & 255)) return PKV_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < pkv_tree_attention_workspace_bytes(num_seqs, d)) return PKV_ERR_WORKSPACE;
  CUtensorMap maps[4];
  if (!get_pool_maps(*pool, &maps[0], &maps[1], 1, 1)) return PKV_ERR_CUDA;
  int rc = make_rows_tensor_map(&maps[2], k_nodes, pool->dtype, d, hkv, total_nodes, k_stride_h, k_stride_n, kNK);
  if (rc == PKV_OK)
    rc = make_rows_tensor_map(&maps[3], v_nodes, pool->dtype, d, hkv, total_nodes, v_stride_h, v_stride_n, kNK);
  if (rc != PKV_OK) return rc;
  TreeParams p;
  p.out = out;
  p.q = q;
  p.cu = cu_nodes;
  p.ctx = context_lens;
  p.mask = reinterpret_cast<const uint64_t*>(mask);
  p.tables = tables->block_tables;
  p.seq_rows = tables->seq_rows;
  p.status = status_dev;
  p.max_units = kWaves * resident(d);
  p.plan = static_cast<int32_t*>(workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan_bytes(num_seqs));
  p.part_o = p.part_ml + (int64_t)p.max_units * 256;
  p.out_st = out_stride_n, p.out_sh = out_stride_h;
  p.q_st = q_stride_n, p.q_sh = q_stride_h;
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
  p.q_vec16 = (addr(q) & 15) == 0 && ((q_stride_n | q_stride_h) & 7) == 0;
  p.out_vec16 = (addr(out) & 15) == 0 && ((out_stride_n | out_stride_h) & 7) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pool->dtype == PKV_F16)
    return d == 64 ? launch<__half, 64>(maps, p, st) : launch<__half, 128>(maps, p, st);
  return d == 64 ? launch<__nv_bfloat16, 64>(maps, p, st) : launch<__nv_bfloat16, 128>(maps, p, st);
}
