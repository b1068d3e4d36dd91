// The steps around tree attention that a speculative decoding step runs on the GPU: block
// tables and slot maps from request lengths, the drafted trees' ancestor masks and
// positions, and the acceptance of a path with its K/V written to the cache. None has a
// counterpart in the reference, which decodes one token per sequence and plans every step
// on the host (engine/kv_cache.py:542-573, 597-609). With these three a step's lengths
// never visit the host: accept_tree advances them where the next extend_tables reads them.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"

namespace pkv {
namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------- block tables from lengths
// For request b (len_b cached tokens, new_b new ones, held_b blocks in its table row):
//   need_b  = max(held_b, ceil((len_b + new_b) / bs)),  fresh_b = need_b - held_b
//   its fresh blocks are free[head + F_b ..], F_b = sum of fresh over earlier requests
//   cu[b]   = sum of new over earlier requests; token t of b sits at position
//             len_b + (t - cu[b]) and slot block(position / bs) * bs + position % bs
// All or nothing: when a request does not fit its row, or the free list is too short, no
// table, held count or head changes and every slot is -1.
//
// Every CTA scans all requests for itself (a few thousand integers, read from L2) and then
// takes its share of the tokens and table entries, so one launch does what a scan kernel and
// a scatter kernel would. What the call costs is latency: a launch, one round of loads, the
// scan's two barriers, a table lookup and the stores. As many CTAs run as the tokens fill (2048
// each). Where outputs continue an input in place, every CTA must have read it first: up to
// 16 K tokens by a cluster's barrier, beyond that by a second launch of one CTA that writes
// them. Measured, apart and in place: 250 requests of one token 3.8 and 4.1 us; 61 requests with
// 8 K tokens 4.5 and 5.0, with 16 K 4.9 and 5.5, with 122 K (2 MB written) 5.1 and 7.8, 15 if one
// cluster took them.
constexpr int kPlanSeqs = 4096;   // requests per call
constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;      // the portable cluster size
constexpr int kPlanTokens = 2 * kPlanThreads;  // tokens of a CTA: two per thread

struct PlanParams {
  int32_t* tables;
  const int32_t* seq_rows;
  const int32_t* lengths;
  const int32_t* new_tokens;
  const int32_t* held;
  const int32_t* free_blocks;
  const int32_t* free_head;
  int32_t* cu;
  int32_t* ctx;
  int64_t* positions;
  int64_t* slots;
  int32_t* held_out;
  int32_t* head_out;
  int32_t* status;
  int64_t table_stride, num_free, total_tokens;
  int32_t rows, cols, batch, bs, shift;  // shift: log2(bs), or -1
  int32_t clustered, writes_map, writes_state;
  // n / bs for 0 <= n < 2^31
  __device__ uint32_t blocks_before(uint32_t n) const { return shift >= 0 ? n >> shift : n / (uint32_t)bs; }
};

// Exclusive prefix sums of two values per thread over the CTA; totals in *ta, *tb.
__device__ inline void block_scan2(int64_t& a, int64_t& b, int64_t* ta, int64_t* tb) {
  __shared__ int64_t wa[32], wb[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) ia += ua, ib += ub;
  }
  if (lane == 31) wa[warp] = ia, wb[warp] = ib;
  __syncthreads();
  if (warp == 0) {
    int64_t xa = lane < nw ? wa[lane] : 0, xb = lane < nw ? wb[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t ua = __shfl_up_sync(0xffffffffu, xa, o), ub = __shfl_up_sync(0xffffffffu, xb, o);
      if (lane >= o) xa += ua, xb += ub;
    }
    if (lane < nw) wa[lane] = xa, wb[lane] = xb;
  }
  __syncthreads();
  *ta = wa[nw - 1];
  *tb = wb[nw - 1];
  a = ia - a + (warp ? wa[warp - 1] : 0);
  b = ib - b + (warp ? wb[warp - 1] : 0);
}

// The last i in [0, n) with first[i] <= x, for non-decreasing first with first[0] <= x.
__device__ inline int last_at_most(const int32_t* first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads, 1) extend_tables_kernel(const PlanParams p) {
  extern __shared__ int32_t plan_smem[];
  const int B = p.batch;
  int32_t* s_len = plan_smem;    // [B] cached tokens
  int32_t* s_held = s_len + B;   // [B] blocks held
  int32_t* s_row = s_held + B;   // [B] table row, -1 = padding
  int32_t* s_cu = s_row + B;     // [B + 1] tokens before request b
  int32_t* s_fp = s_cu + B + 1;  // [B + 1] fresh blocks before request b
  const int tid = threadIdx.x;
  const int per = (B + blockDim.x - 1) / blockDim.x;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  const int64_t head = *p.free_head;
  int64_t sum_new = 0, sum_fresh = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    int row = p.seq_rows ? p.seq_rows[b] : b;
    int64_t len = p.lengths[b], n = p.new_tokens[b], held = p.held[b];
    if (row >= p.rows || n < 0 || (row >= 0 && (len < 0 || held < 0 || held > p.cols))) bad = true;
    n = max(n, (int64_t)0);
    int64_t fresh = 0;
    if (row >= 0) {
      const int64_t end = max(len, (int64_t)0) + n;
      const int64_t need = end < 0x7fffffff - p.bs ? p.blocks_before((uint32_t)(end + p.bs - 1)) : 0x7fffffff;
      if (need > p.cols) bad = true;
      fresh = max(need - held, (int64_t)0);
    }
    s_len[b] = (int32_t)max(len, (int64_t)0);
    s_held[b] = (int32_t)held;
    s_row[b] = row;
    s_cu[b] = (int32_t)n;  // the counts themselves, until what came before is known
    s_fp[b] = (int32_t)min(fresh, (int64_t)0x7fffffff);
    sum_new += n;
    sum_fresh += fresh;
  }
  int64_t pre_new = sum_new, pre_fresh = sum_fresh, total_new, total_fresh;
  block_scan2(pre_new, pre_fresh, &total_new, &total_fresh);
  for (int b = b0; b < b1; ++b) {
    const int64_t n = s_cu[b], fresh = s_fp[b];
    s_cu[b] = (int32_t)min(pre_new, p.total_tokens);
    s_fp[b] = (int32_t)min(pre_fresh, (int64_t)0x7fffffff);
    pre_new += n;
    pre_fresh += fresh;
  }
  if (tid == 0) {
    s_cu[B] = (int32_t)min(total_new, p.total_tokens);
    s_fp[B] = (int32_t)min(total_fresh, (int64_t)0x7fffffff);
  }
  bad = __syncthreads_or(bad || total_new > p.total_tokens || head < 0);
  const bool short_of = !bad && total_fresh > max(p.num_free - head, (int64_t)0);
  const bool ok = !bad && !short_of;
  if (p.clustered) cg::this_cluster().sync();  // every CTA has read the lengths, held counts and the head
  const int rank = blockIdx.x, ctas = gridDim.x;

  if (rank == 0 && p.writes_state) {
    if (tid == 0) {
      if (bad) report(p.status, PKV_ERR_OUT_OF_RANGE);
      if (short_of) report(p.status, PKV_ERR_NO_BLOCKS);
      *p.head_out = (int32_t)(head + (ok ? total_fresh : 0));
      p.cu[B] = s_cu[B];
    }
    for (int b = tid; b < B; b += blockDim.x) {
      p.cu[b] = s_cu[b];
      p.ctx[b] = s_row[b] >= 0 ? s_len[b] + (ok ? s_cu[b + 1] - s_cu[b] : 0) : 0;
      p.held_out[b] = s_held[b] + (ok ? s_fp[b + 1] - s_fp[b] : 0);
    }
  }
  if (!p.writes_map) return;
  const int32_t* fresh_blocks = p.free_blocks + head;
  if (ok) {
    for (int k = rank * blockDim.x + tid; k < (int)total_fresh; k += ctas * blockDim.x) {
      const int b = last_at_most(s_fp, B, k);
      const int32_t blk = fresh_blocks[k];
      if (blk < 0) report(p.status, PKV_ERR_OUT_OF_RANGE);
      p.tables[s_row[b] * p.table_stride + s_held[b] + (k - s_fp[b])] = blk;
    }
  }
  if (!p.positions && !p.slots) return;
  // Two tokens per thread and turn, written as one 16-byte store where the arrays allow it.
  const int used = ok ? s_cu[B] : 0, total = (int)p.total_tokens;
  const bool wide = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
  for (int64_t t0 = 2 * ((int64_t)rank * blockDim.x + tid); t0 < total; t0 += 2 * (int64_t)ctas * blockDim.x) {
    int64_t pos[2] = {0, 0}, slot[2] = {-1, -1};
    int b = t0 < used ? last_at_most(s_cu, B, (int)t0) : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = (int)t0 + e;
      if (t0 + e >= used) break;
      while (s_cu[b + 1] <= t) ++b;  // t is before the batch's end
      if (s_row[b] < 0) continue;
      const uint32_t at = (uint32_t)(s_len[b] + (t - s_cu[b])), col = p.blocks_before(at);
      const int32_t blk = (int)col < s_held[b] ? p.tables[s_row[b] * p.table_stride + col]
                                               : fresh_blocks[s_fp[b] + ((int)col - s_held[b])];
      pos[e] = at;
      if (blk < 0) report(p.status, PKV_ERR_OUT_OF_RANGE);
      else slot[e] = (int64_t)blk * p.bs + (at - col * (uint32_t)p.bs);
    }
    if (wide && t0 + 1 < total) {
      if (p.positions) *reinterpret_cast<longlong2*>(p.positions + t0) = make_longlong2(pos[0], pos[1]);
      if (p.slots) *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
    } else {
      for (int e = 0; e < 2 && t0 + e < total; ++e) {
        if (p.positions) p.positions[t0 + e] = pos[e];
        if (p.slots) p.slots[t0 + e] = slot[e];
      }
    }
  }
}

// ---------------------------------------------------------------- tree metadata
// mask[n] = bits of node n's ancestors and itself, 64 nodes to a word; position =
// context_lens[b] + depth, depth = popcount(mask) - 1. A node's ancestors are gathered by
// pointer doubling in shared memory: after round k a node's mask covers its 2^k nearest
// ancestors and its jump points 2^k up, so a chain of 512 nodes takes 9 rounds instead of 512
// dependent loads. One CTA per tree, one thread per node that the mask has room for. Bound by
// the rounds' barriers and the launch: one tree of 8 nodes 1.9 us, 256 trees of 64 to 256
// nodes (1.8 MB) 3.5 us.
constexpr int kTreeWords = 8;                  // mask words
constexpr int kTreeNodes = 64 * kTreeWords;    // nodes of a tree

template <int WORDS>
__global__ void __launch_bounds__(64 * WORDS)
    tree_metadata_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ cu, int32_t batch,
                         const int32_t* __restrict__ ctx, int64_t total, uint64_t* __restrict__ mask, int32_t words,
                         int64_t* __restrict__ positions, int32_t* status) {
  constexpr int kCap = 64 * WORDS;
  __shared__ uint64_t bits[WORDS][kCap];
  __shared__ int32_t jump[kCap];
  const int b = blockIdx.x, i = threadIdx.x;
  if (b == batch) {  // rows behind the last tree: padding of a captured step
    for (int64_t n = max(cu[batch], 0) + i; n < total; n += kCap) {
      for (int w = 0; w < words; ++w) mask[n * words + w] = 0;
      positions[n] = 0;
    }
    return;
  }
  const int lo = cu[b], hi = cu[b + 1];
  const int64_t at = ctx[b];
  if (lo < 0 || hi < lo || hi > total) {
    if (i == 0) report(status, PKV_ERR_OUT_OF_RANGE);
    return;
  }
  const int all = hi - lo, n = min(all, 64 * words);
  if (all > n && i == 0) report(status, PKV_ERR_OUT_OF_RANGE);
  uint64_t own[WORDS];
  int up = -1;
  if (i < n) {
    up = parents[lo + i];
    if (up < -1 || up >= i) {
      report(status, PKV_ERR_OUT_OF_RANGE);
      up = -1;
    }
  }
#pragma unroll
  for (int w = 0; w < WORDS; ++w) own[w] = w == i / 64 ? 1ull << (i % 64) : 0;
  while (__syncthreads_or(up >= 0)) {  // (the round before has read what this one overwrites)
#pragma unroll
    for (int w = 0; w < WORDS; ++w) bits[w][i] = own[w];
    jump[i] = up;
    __syncthreads();
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) own[w] |= bits[w][up];
      up = jump[up];
    }
  }
  if (i < n) {
    int depth = -1;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      if (w < words) mask[(int64_t)(lo + i) * words + w] = own[w];
      depth += __popcll(own[w]);
    }
    positions[lo + i] = at + depth;
  }
  for (int x = n + i; x < all; x += kCap) {  // nodes the mask has no room for
    for (int w = 0; w < words; ++w) mask[(int64_t)(lo + x) * words + w] = 0;
    positions[lo + x] = at;
  }
}

// ---------------------------------------------------------------- acceptance
// The path of tree b starts at its node 0 (the last token decided); from node c it goes to
// the lowest j with parent[j] = c and draft[j] = target[c], while there is one. Its nodes'
// targets are the step's new tokens, and its K/V rows of every layer move from the nodes'
// buffers to positions len_b, len_b + 1, ... of the sequence.
//
// One cluster per tree: every CTA walks the tree for itself (one warp, 32 candidates a
// step by ballot; a path has a handful of nodes), then copies its share of the layers. The
// copies are all the bytes there are; the walk is a chain of shared-memory reads. Measured:
// one tree over 24 layers 4.3 us; 128 trees over 28 layers of 4 heads of 128 (46 MB read and
// written, in rows of 256 bytes) 15.0 us = 3.1 TB/s, 0.47 of the copy bandwidth: a row is one
// half-warp's, and the walk before it takes 3 us. One flat index over all rows with eight loads
// in flight per thread was slower (20 us).
constexpr int kAcceptThreads = 256;
constexpr int kAcceptWidth = 64;  // longest path

struct AcceptParams {
  const int32_t* tables;
  const int32_t* seq_rows;
  const int32_t* parents;
  const int32_t* cu;
  const int64_t* draft;
  const int64_t* target;
  const void* k_nodes;
  const void* v_nodes;
  void* k_pool;
  void* v_pool;
  const int32_t* lengths;
  int32_t* counts;
  int32_t* path;
  int64_t* tokens;
  int32_t* lengths_out;
  int32_t* status;
  int64_t table_stride, k_sl, k_sn, k_sh, v_sl, v_sn, v_sh, total;
  int32_t rows, cols, batch, width, layers, hkv, d, bs, nbt;
};

template <int EW> struct Bytes;
template <> struct Bytes<8> { using type = uint4; };
template <> struct Bytes<1> { using type = uint16_t; };

template <int EW>
__global__ void __launch_bounds__(kAcceptThreads) accept_tree_kernel(const AcceptParams p) {
  __shared__ int32_t s_parent[kTreeNodes];
  __shared__ int64_t s_draft[kTreeNodes], s_target[kTreeNodes];
  __shared__ int32_t s_path[kAcceptWidth], s_block[kAcceptWidth], s_offset[kAcceptWidth], s_count;
  using V = typename Bytes<EW>::type;
  const int tid = threadIdx.x, lane = tid & 31;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int b = blockIdx.x / ctas;
  int row = p.seq_rows ? p.seq_rows[b] : b;
  const int lo = p.cu[b], hi = p.cu[b + 1], len = p.lengths[b];
  bool bad = row >= p.rows || lo < 0 || hi < lo || hi > p.total || (row >= 0 && len < 0);
  int n = bad || row < 0 ? 0 : hi - lo;
  if (n > kTreeNodes) bad = true, n = kTreeNodes;
  if (bad && tid == 0 && rank == 0) report(p.status, PKV_ERR_OUT_OF_RANGE);
  for (int i = tid; i < n; i += kAcceptThreads) {
    s_parent[i] = p.parents[lo + i];
    s_draft[i] = p.draft[lo + i];
    s_target[i] = p.target[lo + i];
  }
  __syncthreads();
  if (tid < 32) {
    int count = n > 0 ? 1 : 0, cur = 0;
    if (lane == 0) s_path[0] = 0;
    while (count > 0 && count < p.width) {
      const int64_t want = s_target[cur];
      int found = -1;
      for (int j0 = cur + 1; j0 < n && found < 0; j0 += 32) {
        const int j = j0 + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, j < n && s_parent[j] == cur && s_draft[j] == want);
        if (hit) found = j0 + __ffs(hit) - 1;
      }
      if (found < 0) break;
      cur = found;
      if (lane == 0) s_path[count] = cur;
      ++count;
    }
    for (int k = lane; k < count; k += 32) {
      const int64_t col = ((int64_t)len + k) / p.bs;
      int blk = col < p.cols ? p.tables[row * p.table_stride + col] : -1;
      if (blk < 0 || blk >= p.nbt) {
        report(p.status, PKV_ERR_OUT_OF_RANGE);
        blk = -1;
      }
      s_block[k] = blk;
      s_offset[k] = (int)(((int64_t)len + k) % p.bs);
    }
    if (lane == 0) s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  cluster.barrier_arrive();  // this CTA has read the length: lengths_out may be the same buffer
  // Rows to copy (K or V, path node, head): where each starts in layer 0 of its source and of
  // the pool. A thread keeps one vector of a row and takes it through four layers at a time.
  const int per_kind = count * p.hkv, rows = 2 * per_kind, vecs = p.d / EW;
  const int64_t pool_layer = (int64_t)p.nbt * p.hkv * p.bs * p.d;
  const int team = max(1, kAcceptThreads / vecs), in_row = tid % vecs, my_row = tid / vecs;
  for (int x = my_row; x < rows && my_row < team; x += team) {
    const int which = x >= per_kind, r = x - which * per_kind, k = r / p.hkv, h = r - k * p.hkv;
    if (s_block[k] < 0) continue;
    const int64_t node = lo + s_path[k];
    const uint16_t* src = which ? static_cast<const uint16_t*>(p.v_nodes) + node * p.v_sn + h * p.v_sh
                                : static_cast<const uint16_t*>(p.k_nodes) + node * p.k_sn + h * p.k_sh;
    uint16_t* dst = static_cast<uint16_t*>(which ? p.v_pool : p.k_pool) +
                    ((int64_t)s_block[k] * p.hkv + h) * p.bs * p.d + (int64_t)s_offset[k] * p.d;
    const int64_t src_layer = which ? p.v_sl : p.k_sl;
    for (int c = in_row; c < vecs; c += kAcceptThreads) {
      for (int l0 = rank; l0 < p.layers; l0 += 4 * ctas) {
        V v[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (l0 + y * ctas < p.layers) v[y] = *reinterpret_cast<const V*>(src + (l0 + y * ctas) * src_layer + c * EW);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (l0 + y * ctas < p.layers) *reinterpret_cast<V*>(dst + (l0 + y * ctas) * pool_layer + c * EW) = v[y];
      }
    }
  }
  cluster.barrier_wait();
  if (rank == 0) {
    for (int k = tid; k < p.width; k += kAcceptThreads) {
      p.path[(int64_t)b * p.width + k] = k < count ? s_path[k] : -1;
      p.tokens[(int64_t)b * p.width + k] = k < count ? s_target[s_path[k]] : -1;
    }
    if (tid == 0) {
      p.counts[b] = count;
      p.lengths_out[b] = len + count;
    }
  }
}

// A launch of `ctas` CTAs in clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), int ctas, int cluster, int threads, size_t smem, cudaStream_t st,
                           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_extend_tables(const pkv_tables* tables, int32_t num_seqs, const int32_t* lengths,
                                 const int32_t* new_tokens, const int32_t* held_blocks, const int32_t* free_blocks,
                                 int64_t num_free, const int32_t* free_head, int32_t block_size, int32_t* cu_seqlens,
                                 int32_t* context_lens, int64_t* positions, int64_t* slot_mapping, int64_t total_tokens,
                                 int32_t* held_out, int32_t* free_head_out, int32_t* status_dev, pkv_stream_t stream) {
  if (!tables || !free_head || !free_head_out || !cu_seqlens || (!free_blocks && num_free > 0)) return PKV_ERR_INVALID_ARGUMENT;
  if (num_seqs > 0 && (!tables->block_tables || !lengths || !new_tokens || !held_blocks || !context_lens || !held_out))
    return PKV_ERR_INVALID_ARGUMENT;
  if (num_seqs < 0 || block_size <= 0 || num_free < 0 || total_tokens < 0 || total_tokens > 0x7fffffff ||
      num_free > 0x7fffffff || tables->rows < 0 || tables->cols < 0 || tables->stride < 0 ||
      (!tables->seq_rows && tables->rows < num_seqs))
    return PKV_ERR_INVALID_ARGUMENT;
  if (num_seqs > kPlanSeqs) return PKV_ERR_UNSUPPORTED;
  PlanParams p;
  p.tables = const_cast<int32_t*>(tables->block_tables);
  p.seq_rows = tables->seq_rows;
  p.lengths = lengths;
  p.new_tokens = new_tokens;
  p.held = held_blocks;
  p.free_blocks = free_blocks;
  p.free_head = free_head;
  p.cu = cu_seqlens;
  p.ctx = context_lens;
  p.positions = positions;
  p.slots = slot_mapping;
  p.held_out = held_out;
  p.head_out = free_head_out;
  p.status = status_dev;
  p.table_stride = tables->stride;
  p.num_free = num_free;
  p.total_tokens = total_tokens;
  p.rows = tables->rows;
  p.cols = tables->cols;
  p.batch = num_seqs;
  p.bs = block_size;
  p.shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  p.writes_map = p.writes_state = 1;
  const size_t smem = (5 * (size_t)num_seqs + 2) * 4;
  static SmemAttribute attribute;
  const cudaError_t e = attribute.set(reinterpret_cast<const void*>(extend_tables_kernel), (5 * kPlanSeqs + 2) * 4);
  if (e != cudaSuccess) return cuda_status(e);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t tokens = positions || slot_mapping ? total_tokens : 0;
  const int ctas = (int)std::max<int64_t>(1, (tokens + kPlanTokens - 1) / kPlanTokens);
  auto overlaps = [](const void* x, const void* y, int64_t n) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    return a < b + 4 * n && b < a + 4 * n;
  };
  // Whether anything the first CTA writes of the new state is still read by another.
  const int32_t* in[4] = {lengths, new_tokens, held_blocks, free_head};
  const int64_t in_n[4] = {num_seqs, num_seqs, num_seqs, 1};
  int32_t* out[4] = {cu_seqlens, context_lens, held_out, free_head_out};
  const int64_t out_n[4] = {(int64_t)num_seqs + 1, num_seqs, num_seqs, 1};
  bool in_place = false;
  for (int i = 0; i < 4; ++i)
    for (int o = 0; o < 4; ++o) in_place = in_place || overlaps(in[i], out[o], std::max(in_n[i], out_n[o]));
  if (ctas == 1 || (in_place && ctas <= kPlanCtas)) {
    int cluster = 1;
    while (cluster < ctas) cluster *= 2;
    // One CTA of few tokens: no more threads than they and the requests need.
    const int threads = cluster > 1 ? kPlanThreads
                                    : std::min<int>(kPlanThreads, (int)(std::max<int64_t>(num_seqs, (tokens + 1) / 2) + 127) / 128 * 128);
    p.clustered = cluster > 1;
    return cuda_status(launch_cluster(extend_tables_kernel, cluster, cluster, std::max(threads, 128), smem, st, p));
  }
  p.clustered = 0;
  p.writes_state = !in_place;
  extend_tables_kernel<<<std::min(ctas, num_sms()), kPlanThreads, smem, st>>>(p);
  if (!in_place) return launch_status();
  p.writes_map = 0;
  p.writes_state = 1;
  extend_tables_kernel<<<1, kPlanThreads, smem, st>>>(p);
  return launch_status();
}

extern "C" int pkv_build_tree_metadata(const int32_t* parents, const int32_t* cu_nodes, int32_t num_seqs,
                                       const int32_t* context_lens, int64_t total_nodes, int64_t* mask,
                                       int32_t mask_words, int64_t* positions, int32_t* status_dev,
                                       pkv_stream_t stream) {
  if (num_seqs < 0 || total_nodes < 0 || total_nodes > 0x7fffffff || mask_words <= 0) return PKV_ERR_INVALID_ARGUMENT;
  if (mask_words > kTreeWords) return PKV_ERR_UNSUPPORTED;
  if (total_nodes == 0) return PKV_OK;
  if (!parents || !cu_nodes || !mask || !positions || (num_seqs > 0 && !context_lens)) return PKV_ERR_INVALID_ARGUMENT;
  auto kernel = mask_words == 1   ? tree_metadata_kernel<1>
                : mask_words == 2 ? tree_metadata_kernel<2>
                : mask_words <= 4 ? tree_metadata_kernel<4>
                                  : tree_metadata_kernel<8>;
  const int threads = 64 * (mask_words <= 2 ? mask_words : mask_words <= 4 ? 4 : 8);
  kernel<<<num_seqs + 1, threads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      parents, cu_nodes, num_seqs, context_lens, total_nodes, reinterpret_cast<uint64_t*>(mask), mask_words, positions,
      status_dev);
  return launch_status();
}

extern "C" int pkv_accept_tree(const pkv_pool* pool, const pkv_tables* tables, int32_t num_seqs, const int32_t* parents,
                               const int32_t* cu_nodes, int64_t total_nodes, const int64_t* draft_tokens,
                               const int64_t* target_tokens, const void* k_nodes, int64_t k_stride_l, int64_t k_stride_n,
                               int64_t k_stride_h, const void* v_nodes, int64_t v_stride_l, int64_t v_stride_n,
                               int64_t v_stride_h, const int32_t* context_lens, int32_t* counts, int32_t* path,
                               int64_t* tokens, int32_t path_width, int32_t* lengths_out, int32_t* status_dev,
                               pkv_stream_t stream) {
  if (!pool || !pool->k || !pool->v || !tables) return PKV_ERR_INVALID_ARGUMENT;
  if (num_seqs < 0 || total_nodes < 0 || total_nodes > 0x7fffffff || path_width <= 0 || pool->num_layers <= 0 ||
      pool->num_kv_heads <= 0 || pool->head_dim <= 0 || pool->block_size <= 0 || pool->num_blocks_total <= 0 ||
      tables->stride < 0 || (!tables->seq_rows && tables->rows < num_seqs))
    return PKV_ERR_INVALID_ARGUMENT;
  if (pool->dtype != PKV_F16 && pool->dtype != PKV_BF16) return PKV_ERR_UNSUPPORTED;
  if (path_width > kAcceptWidth) return PKV_ERR_UNSUPPORTED;
  if (num_seqs == 0) return PKV_OK;
  if (!tables->block_tables || !cu_nodes || !context_lens || !counts || !path || !tokens || !lengths_out)
    return PKV_ERR_INVALID_ARGUMENT;
  if (total_nodes > 0 && (!parents || !draft_tokens || !target_tokens || !k_nodes || !v_nodes))
    return PKV_ERR_INVALID_ARGUMENT;
  AcceptParams p;
  p.tables = tables->block_tables;
  p.seq_rows = tables->seq_rows;
  p.parents = parents;
  p.cu = cu_nodes;
  p.draft = draft_tokens;
  p.target = target_tokens;
  p.k_nodes = k_nodes;
  p.v_nodes = v_nodes;
  p.k_pool = pool->k;
  p.v_pool = pool->v;
  p.lengths = context_lens;
  p.counts = counts;
  p.path = path;
  p.tokens = tokens;
  p.lengths_out = lengths_out;
  p.status = status_dev;
  p.table_stride = tables->stride;
  p.k_sl = k_stride_l, p.k_sn = k_stride_n, p.k_sh = k_stride_h;
  p.v_sl = v_stride_l, p.v_sn = v_stride_n, p.v_sh = v_stride_h;
  p.total = total_nodes;
  p.rows = tables->rows;
  p.cols = tables->cols;
  p.batch = num_seqs;
  p.width = path_width;
  p.layers = pool->num_layers;
  p.hkv = pool->num_kv_heads;
  p.d = pool->head_dim;
  p.bs = pool->block_size;
  p.nbt = pool->num_blocks_total;
  const uintptr_t addr = reinterpret_cast<uintptr_t>(k_nodes) | reinterpret_cast<uintptr_t>(v_nodes) |
                         reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v);
  if (addr & 1) return PKV_ERR_INVALID_ARGUMENT;
  const int64_t strides = k_stride_l | k_stride_n | k_stride_h | v_stride_l | v_stride_n | v_stride_h | p.d;
  const bool vec16 = (addr & 15) == 0 && (strides & 7) == 0;
  // As many CTAs per tree as have a layer to copy and fit one wave (four of them on an SM):
  // every CTA walks its tree first, about as long as a few layers' copies take. At 28 layers
  // of 4 heads of 128: 1 tree 5.2 us (one CTA 10.0), 74 trees 10.9 (19.5), 128 trees 15.2 with
  // four CTAs each (one 25.3, eight 17.7).
  int cluster = 1;
  while (cluster < 8 && 2 * cluster <= p.layers && 2 * cluster * (int64_t)num_seqs <= 4 * num_sms()) cluster *= 2;
  auto kernel = vec16 ? accept_tree_kernel<8> : accept_tree_kernel<1>;
  return cuda_status(launch_cluster(kernel, num_seqs * cluster, cluster, kAcceptThreads, 0,
                                    reinterpret_cast<cudaStream_t>(stream), p));
}
