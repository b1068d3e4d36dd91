// A mixture-of-experts MLP, router included:
//   out = sum_k w_k * down[e_k] . (silu(gate[e_k] . x) * (up[e_k] . x))
// over the top_k experts e_k with the largest logits router . x, w their softmax.
//
// Few tokens are bound by the touched experts' weights (6 hidden intermediate bytes each, read
// once) and by the chain from the logits to the sum; many by the products.
//
// Up to 8 tokens of few weights: one launch, expert_few_kernel below. Else two or three:
// 1. router_kernel: logits in float32, the choice of experts (exact, see choose()), each choice
//    noted in its expert's list.
// 2. (past kDirectTokens) gather_kernel: each expert's token rows one behind the other.
// 3. expert_kernel: the weights are the 128-row operand A of tcgen05.mma (M), an expert's tokens
//    operand B (N, 16 to 256 of them), so that a decode step's few tokens cost no more than their share
//    of the tensor core's columns. A persistent cooperative grid, one CTA per SM; its items are
//    first every (expert, token tile, weight rows) of gate and up, then every one of down, dealt out
//    in turn. The rings of weight and token stages run on from item to item and from the first
//    product to the second: the weights of down stream in while the activations are still being
//    made, and only the tokens' side waits for them (a counter per token tile). Then the
//    weighted sum over each token's experts, in their order.
// On one B200, captured: 64 tokens of 2048 through 8 of 64 experts of 1024 (bf16, 806 MB of weights) 141 us
// = 5.7 TB/s, 0.87 of the copy bandwidth; 16 tokens of 3584 through 2 of 16 experts of 2368 120 us = 6.0 TB/s;
// 2048 tokens of 2048 through 8 of 64 experts of 768 326 us = 0.48 PFLOP/s (0.63 with down's products taken for both
// halves), bound by what comes into the SMs: a stage of 48 KB for some 500 cycles of products comes at 45 to 52 bytes
// a cycle and SM (L2 at 36 % of its peak, DRAM at 46, tensor cores at 37), and by the 134 MB of float32 products written
// and read back (30 us of sums); 333 tokens of 896 through 4 of 60 experts of 616 67 us and one token of 2048
// through 8 of 64 of 768 25 us, bound by the chain: launches and cold instructions 5 us, logits and choice 4-13,
// first data 4, the wait between the products 3, the last sums 2.
//
// No counterpart in the reference, whose MLP is dense (engine/model.py:254-264).
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "tcgen05.cuh"

namespace pkv {
namespace {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;
constexpr int kKB = 64;            // K elements of a chunk: one 128-byte swizzled row
constexpr int kSlotA = 16384;      // weight bytes of a stage: 32, 64 or 128 rows of 4, 2 or 1 chunks
constexpr int kMaxStages = 16;
constexpr int64_t kMaxItems = 1 << 30;
constexpr int kThreads = 384;      // weight copies, token copies, MMA, finished activations, 8 epilogue warps
constexpr int kRouterTokens = 16;  // tokens of a router CTA
constexpr int kMaxTickets = 1024;  // router groups whose experts are spread over several CTAs
constexpr int kRing = 220 * 1024;  // bytes of the stages
constexpr int64_t kDropBytes = 16 << 20;  // from this size of y on the lines are worth an instruction each (combine())

// What persists between calls, zero outside them; the rest of the workspace is written before it is read.
struct Header {
  int32_t counts[kMaxExperts];   // tokens of each expert
  int32_t tickets[kMaxTickets];  // router CTAs done of each group of tokens
  int32_t arrived;               // CTAs that finished their items
  int32_t left;                  // CTAs that finished
};

struct ExpertParams {
  const void* x;
  const void* router;
  const void* gate_up;
  const void* down;
  Header* head;
  float* logits;    // [tokens][experts]
  float* sizes;     // [tokens][experts at most]: no logit's terms |x_i w_i| sum to more than the largest of a token's
  int32_t* perm;    // [experts][tokens]: an expert's choices, token * top_k + k each
  float* weight;    // [tokens][top_k]
  int32_t* done;    // [token tiles]: row tiles of gate and up that are finished
  void* xs;         // [tokens * top_k][hidden], past kDirectTokens: x by expert
  void* act;        // [2][tokens * top_k][inter], an expert's rows one behind the other: the values rounded, and the rest
  float* y;         // [tokens * top_k][hidden]
  void* out;
  int32_t* status;
  int64_t x_stride, out_stride;
  int tokens, hidden, inter, experts, top_k, renormalize;
  int max_tiles;    // entries of done
  int rows1, rows2; // weight rows of an item (gate and up; down): 32, 64 or 128
  int per1, per2;   // items of a tile
  int tile_n;       // tokens of a tile, at most
  int stages, slot_b;
  int acc_cols;     // columns of an accumulator
  bool in16;        // intermediate is a multiple of 16
  bool direct;      // gate and up's token rows: all of x, or the expert's of xs
  bool drop_y;      // y is dropped from L2 once read
  int rows_x, rows_act;  // token rows of a copy of either product
  uint32_t tmem_cols;
};

// The activations between the two products are held in two halves, the value rounded to T and what the
// rounding left, rounded to T: 16 bits of bfloat16, 22 of float16. Rounded once, the result was 1.4 times as far
// from the exact one as its own rounding puts it, and no longer what up to kFewTokens tokens get. Down's products are
// taken for both, of the same weights: for few tokens the weights' stream hides them. Both halves of an item's
// token rows share a stage where it holds them; else the values have the stage of the weights and the rests the next
// one. Up to kJointRows rows the two halves, a copy's values and then its rests, are the columns of one product, which
// takes no longer, and the epilogue adds them (300 tokens through 8 of 128 experts, up to 32 rows an expert: 235 us,
// 251 by two products); more are summed in the accumulator.
constexpr int kJointRows = 32;
template <typename T>
__device__ __forceinline__ void two_halves(float v, T& high, T& rest) {
  high = Dt<T>::from_f(v);
  const float low = v - Dt<T>::to_f(high);
  rest = Dt<T>::from_f(fabsf(low) < INFINITY ? low : 0.f);  // an infinity's rest would be NaN
}

// Where gate and up's tokens come from: up to kDirectTokens are all loaded for every expert, which takes
// its columns of the accumulator; more are laid out by expert first (gathering four rows a copy cost
// as much as a copy of 32: 503 of a stage's 830 cycles at 64 tokens of 8 in 64 experts).
constexpr int kDirectTokens = 128;

// ---------------------------------------------------------------- router

__device__ __forceinline__ uint32_t order_key(float f) {  // larger is later; NaN last, -0 = 0; never 0
  f += 0.f;
  const uint32_t u = __float_as_uint(f);
  return f != f ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Dt<T>::unpack(w[i]);
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}

// router[e] . x[t] in float64, by a warp (every lane gets it).
template <typename T>
__device__ double exact_logit(const ExpertParams& p, int t, int e) {
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + t * p.x_stride);
  const uint4* w = reinterpret_cast<const uint4*>(static_cast<const T*>(p.router) + (int64_t)e * p.hidden);
  double s = 0;
  const int vecs = p.hidden / 8;
  for (int c0 = threadIdx.x & 31; c0 < vecs; c0 += 32 * 8) {
    uint4 u[8], v[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) u[n] = x[min(c0 + 32 * n, vecs - 1)], v[n] = w[min(c0 + 32 * n, vecs - 1)];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      float a[8], b[8];
      unpack8<T>(u[n], a);
      unpack8<T>(v[n], b);
      if (c0 + 32 * n < vecs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (double)a[i] * (double)b[i];
      }
    }
  }
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// The top_k experts of a token and their weights, by a warp. Lane l holds experts l, l + 32, ... A float32
// logit is off by some part of the sum of its terms' sizes, which large terms that cancel make far more than
// the logit. `border` is twice that part: where the last expert in and the first one out are no further apart
// than it allows, those within that of the border are chosen by their float64 logits, so that the choice does
// not hang on the order of a sum. `sizes`: the token's n sums of sizes; those of rows with an infinity or NaN,
// whose logits are none either, do not count. `exact`: float64 scratch of the warp. Lane k < top_k gets the k-th
// expert and its weight.
template <typename T, int NV>
__device__ void choose(const ExpertParams& p, int t, float border, const float* sizes, int n_sizes, double* exact, int& expert,
                       float& weight) {
  const int lane = threadIdx.x & 31;
  const uint32_t all = 0xffffffffu;
  float v[NV];
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < p.experts ? __ldcg(&p.logits[(int64_t)t * p.experts + e]) : 0.f;
    const float size = e < n_sizes ? __ldcg(&sizes[e]) : 0.f;
    if (size < INFINITY) big = max(big, __float_as_uint(size));
  }
  const float tol = __uint_as_float(__reduce_max_sync(all, big)) * border;
  uint32_t taken = 0;
  int mine_e = 0;
  float mine_v = 0.f, last = 0.f;
  for (int j = 0; j <= p.top_k; ++j) {  // one more than are taken: the first one out
    if (j == p.experts) break;
    uint32_t best = 0;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t k = lane + 32 * i < p.experts && !(taken >> i & 1) ? order_key(v[i]) : 0u;
      if (k > best) best = k, at = lane + 32 * i;
    }
    const uint32_t m = __reduce_max_sync(all, best);
    const int e = __reduce_min_sync(all, best == m ? at : 0x7fffffff);
    const float val = key_value(m);
    if (j == p.top_k) {
      // Finite, unlike and near: infinities and NaN compare false.
      if (tol > 0.f && tol < INFINITY && last - val <= tol) {
        int sure = 0;
        taken = 0;
        uint32_t unsure = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          // One difference for both, so that each expert from the last one in upwards is in one of the sets and no
          // other: a rounded last + tol beside it would leave out an expert that is just there.
          const bool here = lane + 32 * i < p.experts, near = fabsf(v[i] - last) <= tol;
          if (here && !near && order_key(v[i]) > order_key(last)) taken |= 1u << i, ++sure;
          if (here && near) unsure |= 1u << i;
        }
        sure = __reduce_add_sync(all, sure);
        for (int i = 0; i < NV; ++i)
          for (uint32_t b = __ballot_sync(all, unsure >> i & 1); b; b &= b - 1) {
            const int c = 32 * i + __ffs(b) - 1;
            const double s = exact_logit<T>(p, t, c);
            if (lane == 0) exact[c] = s;
          }
        __syncwarp();
        for (int n = sure; n < p.top_k; ++n) {
          double top = -INFINITY;
          int c = 0x7fffffff;
          for (int i = 0; i < NV; ++i)
            if ((unsure & ~taken) >> i & 1) {
              const double s = exact[lane + 32 * i];
              if (c == 0x7fffffff || s > top) top = s, c = lane + 32 * i;
            }
          for (int o = 16; o; o >>= 1) {
            const double s = __shfl_xor_sync(all, top, o);
            const int d = __shfl_xor_sync(all, c, o);
            if (d != 0x7fffffff && (c == 0x7fffffff || s > top || (s == top && d < c))) top = s, c = d;
          }
          if (c == 0x7fffffff) break;  // none left, which the sets rule out
          if (lane == (c & 31)) taken |= 1u << (c >> 5);
        }
        __syncwarp();
        // The taken ones to the lanes 0 .. top_k - 1, in the order of their index.
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const uint32_t b = __ballot_sync(all, taken >> i & 1);
          for (uint32_t left = b; left; left &= left - 1, ++n) {
            const int src = __ffs(left) - 1;
            const float val_c = __shfl_sync(all, v[i], src);
            if (lane == n) mine_e = 32 * i + src, mine_v = val_c;
          }
        }
      }
      break;
    }
    last = val;
    if (lane == (e & 31)) taken |= 1u << (e >> 5);
    if (lane == j) mine_e = e, mine_v = val;
  }
  const bool on = lane < p.top_k;
  const uint32_t top = __reduce_max_sync(all, on ? order_key(mine_v) : 0u);
  const float m = key_value(top);
  float sum = 0.f;
  if (p.renormalize) {
    sum = on ? expf(mine_v - m) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += lane + 32 * i < p.experts ? expf(v[i] - m) : 0.f;
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(all, sum, o);
  expert = mine_e;
  weight = on ? expf(mine_v - m) / sum : 0.f;
}

// A CTA takes kRouterTokens tokens and 16 MT experts at a time by mma.sync (m16n8k16: 16 experts by 8
// tokens, the K order free as below), its warps a part of hidden each; grid y shares out the experts.
// The last CTA of a group of tokens chooses, a warp for a token at a time. 2048 tokens of 2048 in 64
// experts took 38 us by fp32 products.
//
// The same products of |x| and |w| give the sums of the terms' sizes. What a logit may be off: mma.sync lines a
// step's 16 products and the sum so far up to the largest of them, cuts each at 2^-25 of its power of two and the
// result at 2^-23 (seen with products of 2^-20 .. 2^-31 beside 1), 5 2^-23 of the warp's sum of sizes at most; the
// sum over the warps adds 2^-24 for each.
template <typename T, int MT, int NV>
__global__ void __launch_bounds__(MT == 1 ? 512 : 256) router_kernel(const ExpertParams p) {
  constexpr int kWarps = MT == 1 ? 16 : 8, kChoosers = NV > 4 ? 8 : kWarps;
  constexpr int kSteps = MT == 1 ? 4 : 1;  // of 64 elements, whose loads go ahead together
  __shared__ union {
    float part[kWarps][16 * MT][kRouterTokens];
    double exact[kChoosers][32 * NV];
  } s;
  __shared__ float s_size[kWarps][kRouterTokens];
  __shared__ int s_last;
  float size_t0 = 0.f;  // of thread t < kRouterTokens' token: the largest sum so far
  const int group = blockIdx.x, t0 = group * kRouterTokens;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  grid_dep_launch_dependents();  // the next kernel sets itself up, and waits
  // The expert kernel's counters of finished tiles start at zero.
  for (int i = (blockIdx.y * gridDim.x + group) * 32 * kWarps + tid; i < p.max_tiles; i += 32 * kWarps * gridDim.x * gridDim.y)
    p.done[i] = 0;
  const T* col[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) col[j] = static_cast<const T*>(p.x) + min(t0 + 8 * j + g, p.tokens - 1) * p.x_stride;
  auto load16 = [&](uint4 (&to)[2], const T* from, int k) {  // 16 elements, zeros past hidden
    const uint4 zero = make_uint4(0, 0, 0, 0);
    to[0] = k < p.hidden ? *reinterpret_cast<const uint4*>(from + k) : zero;
    to[1] = k + 8 < p.hidden ? *reinterpret_cast<const uint4*>(from + k + 8) : zero;
  };
  for (int e0 = blockIdx.y * 16 * MT; e0 < p.experts; e0 += 16 * MT * gridDim.y) {
    const T* row[MT][2];
    float acc[MT][2][4], sizes[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        row[m][h] = static_cast<const T*>(p.router) + (int64_t)min(e0 + 16 * m + 8 * h + g, p.experts - 1) * p.hidden;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = sizes[m][j][i] = 0.f;
    }
    for (int c = warp * 64; c < p.hidden; c += kWarps * 64 * kSteps) {
      uint4 a[kSteps][MT][2][2], b[kSteps][2][2];
#pragma unroll
      for (int n = 0; n < kSteps; ++n) {
        const int k = c + n * kWarps * 64 + q * 16;
#pragma unroll
        for (int m = 0; m < MT; ++m) load16(a[n][m][0], row[m][0], k), load16(a[n][m][1], row[m][1], k);
        load16(b[n][0], col[0], k), load16(b[n][1], col[1], k);
      }
#pragma unroll
      for (int n = 0; n < kSteps; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 &lo = a[n][m][0][h], &hi = a[n][m][1][h];
            constexpr uint32_t kAbs = 0x7fff7fffu;
            const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
            const uint32_t s0[4] = {lo.x & kAbs, hi.x & kAbs, lo.y & kAbs, hi.y & kAbs};
            const uint32_t s1[4] = {lo.z & kAbs, hi.z & kAbs, lo.w & kAbs, hi.w & kAbs};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4& x = b[n][j][h];
              mma16816<T>(acc[m][j], a0, x.x, x.y);
              mma16816<T>(acc[m][j], a1, x.z, x.w);
              mma16816<T>(sizes[m][j], s0, x.x & kAbs, x.y & kAbs);
              mma16816<T>(sizes[m][j], s1, x.z & kAbs, x.w & kAbs);
            }
          }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s.part[warp][16 * m + g + 8 * (i >> 1)][8 * j + 2 * q + (i & 1)] = acc[m][j][i];
    // The largest of the warp's sums for each token: their sum over the warps is no less than any expert's.
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float most = 0.f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = k; i < 4; i += 2) most = sizes[m][j][i] < INFINITY ? fmaxf(most, sizes[m][j][i]) : most;
        for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (g == 0) s_size[warp][8 * j + 2 * q + k] = most;
      }
    __syncthreads();
    for (int i = tid; i < 16 * MT * kRouterTokens; i += 32 * kWarps) {
      const int e = i % (16 * MT), t = i / (16 * MT);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) sum += s.part[k][e][t];
      if (e0 + e < p.experts && t0 + t < p.tokens) p.logits[(int64_t)(t0 + t) * p.experts + e0 + e] = sum;
    }
    if (tid < kRouterTokens) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) sum += s_size[k][tid];
      size_t0 = fmaxf(size_t0, sum);
      if (t0 + tid < p.tokens) p.sizes[(int64_t)(t0 + tid) * p.experts + blockIdx.y] = size_t0;
    }
    __syncthreads();
  }
  if (gridDim.y > 1) {
    if (tid == 0) {
      const bool last = atom_add_acq_rel_gpu(&p.head->tickets[group], 1) == (int)gridDim.y - 1;
      if (last) st_relaxed_gpu(&p.head->tickets[group], 0);
      s_last = last;
    }
    __syncthreads();
    if (!s_last) return;
  }
  // Twice what a logit may be off, a hundredth for the sums of sizes, which are rounded too.
  const float border = 0x1.03p-22f * (5.f * 4 * ((p.hidden + 64 * kWarps - 1) / (64 * kWarps)) + 0.5f * kWarps);
  for (int t = t0 + warp; warp < kChoosers && t < min(t0 + kRouterTokens, p.tokens); t += kChoosers) {
    int e;
    float w;
    choose<T, NV>(p, t, border, p.sizes + (int64_t)t * p.experts, gridDim.y, s.exact[warp], e, w);
    if (lane < p.top_k) {
      const int a = t * p.top_k + lane;
      p.weight[a] = w;
      // Places are handed out in no fixed order: a row's products do not depend on its place.
      p.perm[(int64_t)e * p.tokens + atomicAdd(&p.head->counts[e], 1)] = a;
    }
  }
}

// ---------------------------------------------------------------- experts

// As mbar_wait_until, with the clock read every 64th poll.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, uint64_t deadline) {
  for (int i = 1; !mbar_try_wait(bar, parity); ++i)
    if ((i & 63) == 0 && global_ns() > deadline) return false;
  return true;
}

// The same by a converged warp, in a loop that is one way for all of it.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, uint64_t deadline) {
  for (int i = 1; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++i)
    if ((i & 63) == 0 && __any_sync(0xffffffffu, global_ns() > deadline)) return false;
  return true;
}

struct Item {
  bool second;            // down; else gate and up
  int tile, e, n0, n;     // token tile, its expert, its first and number of tokens
  int row;                // row tile
  int chunks;             // of 64 elements of K
  int halves;             // what becomes of the two halves of its token rows
};
// Gate and up's rows have none; down's are copied and multiplied one behind the other, jointly (a copy brings both,
// one product has both as columns), or the rests in a stage of their own.
enum { kNone, kBoth, kJoint, kSplit };

struct Shared {
  uint64_t full[kMaxStages];   // a stage's weight rows and token rows landed
  uint64_t freed[kMaxStages];  // its MMAs completed
  uint64_t acc_full[2], acc_empty[2], mma_done;
  uint32_t tmem;
  int stored[8];                // items of gate and up whose activations each epilogue warp has stored
  int last;
  int offset[kMaxExperts + 1];  // rows of act before each expert's
  int tile[kMaxExperts + 1];    // token tiles before each expert's
};

// Rows and token tiles before each expert's, by a warp.
__device__ __forceinline__ void scan_experts(const ExpertParams& p, int* offset, int* tile) {
  const int lane = threadIdx.x & 31;
  int rows = 0, tiles = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int c = e0 + lane < p.experts ? __ldcg(&p.head->counts[e0 + lane]) : 0;
    const int own = (c + p.tile_n - 1) / p.tile_n;
    int r = c, n = own;
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) r += a, n += b;
    }
    if (e0 + lane < p.experts) offset[e0 + lane] = rows + r - c, tile[e0 + lane] = tiles + n - own;
    rows += __shfl_sync(0xffffffffu, r, 31);
    tiles += __shfl_sync(0xffffffffu, n, 31);
  }
  if (lane == 0) offset[p.experts] = rows, tile[p.experts] = tiles;
}

// x's rows by expert. A warp copies a row at a time; bound by the rows' bytes.
__global__ void __launch_bounds__(256) gather_kernel(const ExpertParams p) {
  __shared__ int offset[kMaxExperts + 1], tile[kMaxExperts + 1];
  grid_dep_launch_dependents();
  grid_dep_wait();
  if (threadIdx.x < 32) scan_experts(p, offset, tile);
  __syncthreads();
  const int rows = p.tokens * p.top_k, lane = threadIdx.x & 31, vecs = p.hidden / 8;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
    int lo = 0, hi = p.experts - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (offset[mid] <= r) lo = mid; else hi = mid - 1;
    }
    const int t = p.perm[(int64_t)lo * p.tokens + r - offset[lo]] / p.top_k;
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + t * p.x_stride);
    uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.xs) + (int64_t)r * p.hidden);
#pragma unroll 8
    for (int c = lane; c < vecs; c += 32) to[c] = __ldg(from + c);
  }
}

// Item i, by a converged warp; false past the last. Not inlined: the roles share its instructions, which
// a launch has to fetch anew (they took 6000 cycles before the first copy when each role had its own).
__device__ __noinline__ bool find_item(const ExpertParams& p, const Shared& s, int i, Item& it) {
  const int lane = threadIdx.x & 31, first = s.tile[p.experts] * p.per1;
  it.second = i >= first;
  const int per = it.second ? p.per2 : p.per1;
  if (it.second) i -= first;
  it.tile = i / per, it.row = i - it.tile * per;
  if (it.second && it.tile >= s.tile[p.experts]) return false;
  it.chunks = ((it.second ? p.inter : p.hidden) + kKB - 1) / kKB;
  // The last expert whose tiles start at or before it.tile, among 32 marks and then between two.
  const int stride = (p.experts + 31) / 32;
  int at = lane * stride;
  const int mark = (__popc(__ballot_sync(0xffffffffu, at < p.experts && s.tile[at] <= it.tile)) - 1) * stride;
  at = mark + lane;
  it.e = mark + __popc(__ballot_sync(0xffffffffu, lane < stride && at < p.experts && s.tile[at] <= it.tile)) - 1;
  // An expert's tiles are alike: one full and one of a few tokens would take SMs unequal times.
  const int count = s.offset[it.e + 1] - s.offset[it.e], tiles = s.tile[it.e + 1] - s.tile[it.e];
  const int size = ((count + tiles - 1) / tiles + 15) & ~15;  // at most tile_n, a multiple of 16: no tile is empty
  // Of all of an expert's tiles alike, by their size and not by their rows: which rows the last, smaller tile has is a
  // matter of timing, and the order of their sums must not be.
  const bool hold = 2 * ((size + p.rows_act - 1) / p.rows_act * p.rows_act) * 128 * (128 / p.rows2) <= p.slot_b;  // in one stage
  it.halves = !it.second ? kNone : !hold ? kSplit : size <= kJointRows ? kJoint : kBoth;
  it.n0 = (it.tile - s.tile[it.e]) * size;
  it.n = min(size, count - it.n0);
  return true;
}

// Every CTA of the grid has come here `times` times; what it wrote before is visible.
__device__ __forceinline__ void grid_barrier(const ExpertParams& p, int times, uint64_t deadline = 0) {
  __syncthreads();
  if (threadIdx.x == 0) {
    atom_add_acq_rel_gpu(&p.head->arrived, 1);
    const uint64_t end = max(deadline, (uint64_t)global_ns()) + 2 * kWaitBudgetNs;  // past the waits of every CTA
    for (int n = 1; ld_acquire_gpu(&p.head->arrived) < times * (int)gridDim.x; ++n)
      if ((n & 63) == 0 && global_ns() > end) {
        report(p.status, PKV_ERR_TIMEOUT);
        break;
      }
  }
  __syncthreads();
}

// 128 bytes that nothing reads any more: not written back to memory, where they still lie in L2.
__device__ __forceinline__ void drop_line(const void* line) { asm volatile("discard.global.L2 [%0], 128;" ::"l"(line) : "memory"); }

// 32 bytes in one load: by two of 16 a warp would ask L2 for every 32-byte sector twice.
__device__ __forceinline__ void load8(float (&v)[8], const float* from) {
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(from)
               : "memory");
}

// out = the sum over each token's experts, in their order, of its products; by the whole grid. Eight
// products' loads go ahead together. A large y would be written to memory from L2 while it is read, and after:
// its lines are dropped instead (134 MB at 2048 tokens: 274 us with them written, 267 without; the same for xs
// behind its last reader took 5 us more).
template <typename T>
__device__ __forceinline__ void combine(const ExpertParams& p, const float* weight) {
  const int per_row = p.hidden / 8;
  const uint32_t at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  const int step_t = step / per_row, step_c = step % per_row;
  for (int t = at / per_row, u = at % per_row; t < p.tokens; t += step_t, u += step_c) {
    if (u >= per_row) {
      u -= per_row;
      if (++t >= p.tokens) break;
    }
    const int c = u * 8;
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    for (int k0 = 0; k0 < p.top_k; k0 += 8) {
      float v[8][8], w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int a = t * p.top_k + min(k0 + k, p.top_k - 1);
        load8(v[k], p.y + (int64_t)a * p.hidden + c);
        w[k] = weight[a];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < p.top_k)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += w[k] * v[k][e];
    }
    uint4 o;
    o.x = Dt<T>::pack(sum[0], sum[1]), o.y = Dt<T>::pack(sum[2], sum[3]);
    o.z = Dt<T>::pack(sum[4], sum[5]), o.w = Dt<T>::pack(sum[6], sum[7]);
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + t * p.out_stride + c) = o;
    if (p.drop_y) {  // a line of a product is four lanes'
      __syncwarp(0xfu << (threadIdx.x & 28));
      if ((u & 3) == 0)
        for (int k = 0; k < p.top_k; ++k) drop_line(p.y + (int64_t)(t * p.top_k + k) * p.hidden + c);
    }
  }
}

// The last CTA to come here leaves the workspace ready for the next call.
__device__ __forceinline__ void leave(const ExpertParams& p, int* s_last) {
  if (threadIdx.x == 0) *s_last = atom_add_acq_rel_gpu(&p.head->left, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (*s_last) {
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x) p.head->counts[e] = 0;
    if (threadIdx.x == 0) p.head->arrived = p.head->left = 0;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    expert_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_gu,
                  const __grid_constant__ CUtensorMap map_act, const __grid_constant__ CUtensorMap map_down,
                  const __grid_constant__ CUtensorMap map_x128, const __grid_constant__ CUtensorMap map_act128,
                  const __grid_constant__ CUtensorMap map_halves,
                  const __grid_constant__ ExpertParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared s;
  uint8_t* ring_a = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring_b = ring_a + p.stages * kSlotA;
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const int G = gridDim.x;

  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&s.full[i], 2);
      mbar_init(&s.freed[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], 8);
    }
    mbar_init(&s.mma_done, 1);
    for (int i = 0; i < 8; ++i) s.stored[i] = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_gu);
    prefetch_tensormap(&map_act);
    prefetch_tensormap(&map_down);
  }
  if (warp == 2) {
    tmem_alloc(&s.tmem, p.tmem_cols);
    tc_fence_before_sync();
  }
  grid_dep_wait();
  if (warp == 1) scan_experts(p, s.offset, s.tile);
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s.tmem;
  // Past the time that the kernel's own work takes (4 us a chunk and CTA are four times what it does).
  const int64_t chunks = (int64_t)s.tile[p.experts] * ((int64_t)p.per1 * (p.hidden / kKB + 1) + (int64_t)p.per2 * (p.inter / kKB + 1));
  const uint64_t deadline = global_ns() + kWaitBudgetNs + (uint64_t)(chunks / G) * 4000;
  Item it;
  bool ok = true;

  if (warp == 0 || warp == 1) {
    // ---------------------------------------------------------------- copies: weights, tokens
    // The whole warp runs the loop and one lane issues: a copy's operands are uniform registers, and
    // in a branch of one lane each would be moved there anew for every copy.
    const bool weights = warp == 0;
    // Weights pass through L2 even where an expert has several token tiles: those run at about the same
    // time (kept in L2 for them, 333 tokens took 61 us instead of 59, 2048 tokens 285 instead of 282).
    const uint64_t once = policy_evict_first(), reused = policy_evict_last();
    const bool leader = elect_one();
    int issued = 0, slot = 0;
    uint32_t round = 0;  // of the ring
    for (int i = blockIdx.x; ok && __all_sync(0xffffffffu, find_item(p, s, i, it)); i += G) {
      const bool second = uniform(it.second);
      const int e = uniform(it.e), rows = second ? p.rows2 : p.rows1, wide = 128 / rows;
      const int k1 = uniform(it.chunks), pad = uniform((it.n + 15) & ~15);
      const int row = uniform(it.row) * (second ? p.rows2 : p.rows1 / 2), box = second ? p.rows2 : 32;
      const bool direct = !second && p.direct;
      const int first = direct ? 0 : uniform(s.offset[it.e] + it.n0), columns = direct ? p.tile_n : pad;
      const int rows_b = second ? p.rows_act : p.rows_x, loaded = (columns + rows_b - 1) / rows_b * rows_b;
      if (!weights && second) {  // the tile's activations
        if (lane == 0)
          for (int n = 1; ld_acquire_gpu(&p.done[it.tile]) < p.per1; ++n)
            if ((n & 63) == 0 && global_ns() > deadline) {
              ok = false;
              break;
            }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_proxy_async_global();
      }
      const int how = uniform(it.halves);
      const bool joint = how == kJoint;
      const CUtensorMap* map_w = second ? &map_down : &map_gu;
      const CUtensorMap* map_b = joint ? &map_halves : second ? &map_act : &map_x;
      const CUtensorMap* map_b128 = second ? &map_act128 : &map_x128;
      const int stack = second ? e : 2 * e;
      // Stages of a step, and the halves of one that are copied one after another; a joint copy brings both.
      const int parts = how == kSplit ? 2 : 1, halves = how == kBoth ? 2 : 1, twice = joint ? 2 : 1;
      for (int ks = 0; ok && ks < k1; ks += wide)
        for (int part = 0; part < parts; ++part) {
          if (round > 0 && !wait_warp(&s.freed[slot], (round - 1) & 1, deadline)) {
            ok = false;
            break;
          }
          uint64_t* bar = &s.full[slot];
          const int chunks = min(wide, k1 - ks);
          if (weights) {
            uint8_t* dst = ring_a + slot * kSlotA;
            const int fresh = part ? 0 : chunks;  // none for the rests: those of the stage before
            if (leader) mbar_arrive_expect_tx(bar, fresh * rows * 128);
            for (int c = 0; c < fresh; ++c, dst += rows * 128) {
              if (second || !p.in16) {
                for (int b = 0; b < rows; b += box)
                  if (leader)
                    tma_load_4d(dst + b * 128, map_w, (ks + c) * kKB, row + (second ? b : b / 2), stack, 0, bar, once);
              } else {
                if (leader) tma_load_4d(dst, map_w, (ks + c) * kKB, 0, stack, row / 16, bar, once);
              }
            }
          } else {
            uint8_t* dst = ring_b + slot * p.slot_b;
            if (leader) mbar_arrive_expect_tx(bar, chunks * halves * twice * loaded * 128);
            for (int c = 0; c < chunks; ++c)
              for (int h = part; h < part + halves; ++h)
                for (int b = 0; b < columns;) {
                  // A copy takes this warp some 50 cycles whatever its rows: 128 at once where they are there to read.
                  const bool many = rows_b == 32 && columns - b > 96;
                  const int copied = many ? 128 : rows_b;
                  if (leader) tma_load_4d(dst, many ? map_b128 : map_b, (ks + c) * kKB, first + b, h, 0, bar, reused);
                  b += copied, dst += copied * twice * 128;
                }
          }
          ++issued;
          if (++slot == p.stages) slot = 0, ++round;
        }
    }
    if (!ok && lane == 0) {  // this warp's copies have landed before its CTA may leave
      report(p.status, PKV_ERR_TIMEOUT);
      const uint64_t end = global_ns() + kWaitBudgetNs / 4;
      for (int q = max(0, issued - p.stages); q < issued; ++q) wait_for(&s.full[q % p.stages], (q / p.stages) & 1, end);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------------------------------------------------------- MMA issue
    constexpr bool kBf16 = Dt<T>::code == PKV_BF16;
    const bool leader = elect_one();
    const uint64_t a0 = umma_desc_sw128(smem_u32(ring_a), 16, 1024), b0 = umma_desc_sw128(smem_u32(ring_b), 16, 1024);
    int c = 0, slot = 0;
    uint32_t round = 0;
    for (int i = blockIdx.x; ok && __all_sync(0xffffffffu, find_item(p, s, i, it)); i += G, ++c) {
      const bool second = uniform(it.second);
      const int b = c & 1;
      if (c >= 2 && !wait_warp(&s.acc_empty[b], ((c >> 1) - 1) & 1, deadline)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const int rows = second ? p.rows2 : p.rows1, wide = 128 / rows;
      const int k1 = uniform(it.chunks), pad = uniform((it.n + 15) & ~15);
      const int columns = !second && p.direct ? p.tile_n : pad;
      const int rows_b = second ? p.rows_act : p.rows_x, loaded = (columns + rows_b - 1) / rows_b * rows_b;
      const int how = uniform(it.halves);
      const bool joint = how == kJoint;
      const int parts = how == kSplit ? 2 : 1, halves = how == kBoth ? 2 : 1, twice = joint ? 2 : 1;
      const uint32_t idesc = umma_idesc_f16(kBf16, false, 128, joint ? 2 * loaded : columns);
      const uint32_t d = tmem + (uint32_t)(b * p.acc_cols);
      bool more = false;
      for (int ks = 0; ok && ks < k1; ks += wide) {
        // An item of fewer than 128 weight rows reads on into what is behind them: those lanes of the
        // accumulator are not read. Descriptors count in 16 bytes.
        const uint64_t ad = a0 + slot * (kSlotA >> 4);
        const int with_weights = slot, chunks = min(wide, k1 - ks);
        for (int part = 0; part < parts; ++part) {
          if (!wait_warp(&s.full[slot], round & 1, deadline)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          uint64_t bd = b0 + (uint32_t)(slot * (p.slot_b >> 4));
          for (int n = 0; n < chunks; ++n)
            for (int h = 0; h < halves; ++h, bd += loaded * twice * 8) {
              umma_f16_ss_x4(leader, d, ad + n * rows * 8, bd, idesc, more);
              more = true;
            }
          // The weights' stage is free once the rests in the next one are multiplied.
          if (leader && part == parts - 1) umma_commit(&s.freed[with_weights]);
          if (leader && part) umma_commit(&s.freed[slot]);
          if (++slot == p.stages) slot = 0, ++round;
        }
      }
      if (ok && leader) umma_commit(&s.acc_full[b]);
    }
    if (leader) {
      if (!ok) report(p.status, PKV_ERR_TIMEOUT);
      umma_commit(&s.mma_done);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ---------------------------------------------------------------- finished activations
    // A fence takes 8 to 12 thousand cycles behind the weights' stream: the epilogue does not wait for it.
    int ready = 0;  // items that every epilogue warp has stored, and that the fence covers
    int n = 0;
    for (int i = blockIdx.x; ok && find_item(p, s, i, it) && !it.second; i += G, ++n) {
      if (n >= ready) {
        for (int k = 1; ok; ++k) {
          ready = (int)__reduce_min_sync(0xffffffffu, lane < 8 ? (unsigned)ld_acquire_cta(&s.stored[lane]) : 0x7fffffffu);
          if (ready > n) break;
          if ((k & 63) == 0) ok = __all_sync(0xffffffffu, global_ns() <= deadline);
        }
        if (!ok) break;
        __syncwarp();
        fence_proxy_async_global();  // the rows are read by bulk copies
        fence_acq_rel_gpu();
      }
      if (lane == 0) atom_add_acq_rel_gpu(&p.done[it.tile], 1);
    }
    if (!ok && lane == 0) report(p.status, PKV_ERR_TIMEOUT);
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- epilogue
    // Two warps a lane quarter, each every other 16 columns. A block of columns is read while the last
    // one is worked on, and the accumulator is given back once the last block has been read.
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t tl = tmem + ((uint32_t)(q * 32) << 16);
    const bool low = lane < 16;
    T* act = static_cast<T*>(p.act);
    int c = 0;
    for (int i = blockIdx.x; find_item(p, s, i, it); i += G, ++c) {
      const int b = c & 1;
      const bool second = it.second, direct = !second && p.direct;
      const int n = q * 32 < (second ? p.rows2 : p.rows1) ? it.n : 0;  // columns to finish
      int list[8];  // the choices of this warp's columns, lane l & 15 of each block
      if (second || direct) {
        const int32_t* perm = p.perm + (int64_t)it.e * p.tokens + it.n0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = 16 * (2 * j + half) + (lane & 15);
          list[j] = col < n ? __ldg(&perm[col]) : 0;
          if (direct) list[j] /= p.top_k;
        }
      }
      // Gate and up: lanes 0 .. 15 hold gate rows, 16 .. 31 the same up rows; of two columns a lane finishes one.
      const int r = second ? it.row * p.rows2 + q * 32 + lane : it.row * (p.rows1 / 2) + q * 16 + (lane & 15);
      const bool in = r < (second ? p.hidden : p.inter);
      T *to_act = act + (int64_t)(s.offset[it.e] + it.n0) * p.inter + r, *to_rest = to_act + (int64_t)p.tokens * p.top_k * p.inter;
      float* to_y = p.y + r - (lane & 3);  // the first of four rows: hidden is a multiple of 8
      // After a wait that ran out the warp goes on to its barriers, without data: the others wait there.
      ok = ok && wait_for(&s.acc_full[b], (c >> 1) & 1, deadline);
      tc_fence_after_sync();
      const uint32_t d = tl + (uint32_t)(b * p.acc_cols);
      const bool joint = it.halves == kJoint;  // then a warp has one block of columns at most
      uint32_t v[2][16];
      auto fetch = [&](int j) {
        if (direct) {  // the columns of the tokens themselves
#pragma unroll
          for (int k = 0; k < 16; ++k) v[j & 1][k] = tmem_ld1(d + __shfl_sync(0xffffffffu, list[j], k));
        } else {
          tmem_ld16(d + 16 * (2 * j + half), v[j & 1]);
        }
      };
      if (joint && 16 * half < n) {  // the columns of a copy's values, then of its rests
        const int at = 16 * half / p.rows_act * 2 * p.rows_act + 16 * half % p.rows_act;
        tmem_ld16(d + at, v[0]);
        tmem_ld16(d + at + p.rows_act, v[1]);
      } else if (16 * half < n) {
        fetch(0);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c0 = 16 * (2 * j + half);
        if (c0 >= n) break;
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) asm volatile("" : "+r"(v[j & 1][k]));  // read from here on
        if (j == 0 && joint) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            asm volatile("" : "+r"(v[1][k]));
            v[0][k] = __float_as_uint(__uint_as_float(v[0][k]) + __uint_as_float(v[1][k]));
          }
        }
        if (j < 7 && c0 + 32 < n) fetch(j + 1);
        if (j == 7 || c0 + 32 >= n) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.acc_empty[b]);
        }
        if (second) {
#pragma unroll
          for (int k = 0; k < 16; k += 4) {  // four rows of four columns turned about: 16 bytes of one column a lane
            uint32_t* x = &v[j & 1][k];
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? x[h] : x[h + 1], 1);
              x[h] = lane & 1 ? other : x[h], x[h + 1] = lane & 1 ? x[h + 1] : other;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 2 ? x[h] : x[h + 2], 2);
              x[h] = lane & 2 ? other : x[h], x[h + 2] = lane & 2 ? x[h + 2] : other;
            }
            const int at = __shfl_sync(0xffffffffu, list[j], k + (lane & 3));
            if (c0 + k + (lane & 3) < n && in)
              *reinterpret_cast<uint4*>(to_y + (int64_t)at * p.hidden) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const uint32_t x = v[j & 1][k], y = v[j & 1][k + 1];
            const float other = __uint_as_float(__shfl_xor_sync(0xffffffffu, low ? y : x, 16));
            const float g = low ? __uint_as_float(x) : other;
            const float u = low ? other : __uint_as_float(y);
            const int col = c0 + k + (low ? 0 : 1);
            if (in && col < n) {
              const int64_t at = (int64_t)col * p.inter;
              two_halves(__fdividef(g, 1.f + __expf(-g)) * u, to_act[at], to_rest[at]);
            }
          }
        }
      }
      if (16 * half >= n) {  // nothing of this tile
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.acc_empty[b]);
      }
      if (!second) {
        __syncwarp();
        if (lane == 0) st_release_cta(&s.stored[warp - 4], c + 1);
      }
    }
    if (!ok && lane == 0) report(p.status, PKV_ERR_TIMEOUT);
  }
  __syncthreads();
  if (warp == 2) {
    if (!wait_for(&s.mma_done, 0, global_ns() + kWaitBudgetNs) && lane == 0) report(p.status, PKV_ERR_TIMEOUT);
    tc_fence_after_sync();
    tmem_dealloc(tmem, p.tmem_cols);
  }

  grid_barrier(p, 1, deadline);
  combine<T>(p, p.weight);
  leave(p, &s.last);
}

// ---------------------------------------------------------------- experts, few tokens

// Up to kFewTokens tokens, in one launch with the router: the latency of a decode step of one request.
//
// A unit is 16 weight rows by an expert's tokens (the 8 columns of mma.sync m16n8k16), and a warp's own.
// The warp streams its units' rows through a ring of its own in shared memory by cp.async, kDepth - 1
// chunks ahead of the products, on from unit to unit and from gate and up to down: no CTA-wide step
// but the grid's barriers. A chunk has 512 bytes of each row: 256 cost 4 to 25 percent, 128 30 to 70.
// Teams of two or four warps to a unit, a part of K each, won 6 percent and lost 10 as often. Rows
// 0 .. 7 of a unit are gate and 8 .. 15 the same up rows, so that a thread holds both. The K order of a
// product is free: a lane takes 16 consecutive elements of its rows, and of its token.
constexpr int kFewTokens = 8;
constexpr int kFewChoices = kFewTokens * kMaxTopK;
constexpr int kFewThreads = 256;
constexpr int kDepth = 3;
constexpr int kChunkK = 256;                // elements of a row in a chunk
constexpr int kChunk = 16 * kChunkK * 2;  // bytes: 16 rows
constexpr int kFewSmem = kFewThreads / 32 * kDepth * kChunk;

struct FewShared {
  float part[8][kFewTokens];       // a logit's parts, by warp
  float size[8][kFewTokens];       // and those of its terms' sizes
  float weight[kFewChoices];       // of each choice, token * top_k + k
  alignas(16) int expert[kFewChoices];
  uint32_t lead[kFewChoices / 32]; // choices that are their expert's first
  int group_e[kFewChoices];        // the chosen experts
  int group_n[kFewChoices];        // their tokens' number
  int group_a[kFewChoices][kFewTokens];  // and choices
  int last;
};

// Where a warp's copies are: its unit of which product, and the chunk.
template <typename T>
struct Copies {
  const T* low;         // row 0
  int64_t high;         // from row 0 to row 8
  int second, u, k, K;  // u past the last unit: none left
};

__device__ __forceinline__ void cp_async_16_or_0(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Logits of every expert, an expert per CTA at a time, its warps a part of hidden each.
template <typename T>
__device__ __forceinline__ void few_logits(const ExpertParams& p, FewShared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, vecs = p.hidden / 8;
  for (int e = blockIdx.x; e < p.experts; e += gridDim.x) {
    float acc[kFewTokens], size[kFewTokens];
#pragma unroll
    for (int t = 0; t < kFewTokens; ++t) acc[t] = size[t] = 0.f;
    const uint4* w = reinterpret_cast<const uint4*>(static_cast<const T*>(p.router) + (int64_t)e * p.hidden);
    for (int c = threadIdx.x; c < vecs; c += kFewThreads) {
      float a[8], b[8];
      unpack8<T>(w[c], a);
#pragma unroll
      for (int t = 0; t < kFewTokens; ++t)
        if (t < p.tokens) {
          unpack8<T>(reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + t * p.x_stride)[c], b);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[t] += a[i] * b[i], size[t] += fabsf(a[i]) * fabsf(b[i]);
        }
    }
#pragma unroll
    for (int t = 0; t < kFewTokens; ++t) {
      if (t < p.tokens)
        for (int o = 16; o; o >>= 1) {
          acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
          size[t] += __shfl_xor_sync(0xffffffffu, size[t], o);
        }
      if (lane == 0) s.part[warp][t] = acc[t], s.size[warp][t] = size[t];
    }
    __syncthreads();
    if (threadIdx.x < p.tokens) {
      float sum = 0.f, size_sum = 0.f;
      for (int k = 0; k < kFewThreads / 32; ++k) sum += s.part[k][threadIdx.x], size_sum += s.size[k][threadIdx.x];
      p.logits[(int64_t)threadIdx.x * p.experts + e] = sum;
      p.sizes[(int64_t)threadIdx.x * p.experts + e] = size_sum;
    }
    __syncthreads();
  }
}

// Every CTA chooses for all tokens, a warp each, and lists the chosen experts in the order of their first
// choice: the same lists everywhere. Returns their number.
template <typename T, int NV>
__device__ __forceinline__ int few_groups(const ExpertParams& p, FewShared& s, double* exact) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = p.tokens * p.top_k;
  if (tid < kFewChoices) s.expert[tid] = -1;
  __syncthreads();
  if (warp < p.tokens) {
    int e;
    float w;
    // A thread's terms, five steps of shuffles and eight warps: 2^-24 of the sum of sizes for each addition. Twice
    // that, and a hundredth for the sums of sizes.
    const float border = 0x1.03p-23f * (8.f * ((p.hidden / 8 + kFewThreads - 1) / kFewThreads) + 13.f);
    choose<T, NV>(p, warp, border, p.sizes + (int64_t)warp * p.experts, p.experts, exact + warp * kMaxExperts, e, w);
    if (lane < p.top_k) s.expert[warp * p.top_k + lane] = e, s.weight[warp * p.top_k + lane] = w;
  }
  __syncthreads();
  int first = -1, rank = 0, count = 0;
  const int mine = tid < n ? s.expert[tid] : -2;
  if (tid < kFewChoices) {
    for (int a = 0; a < n; a += 4) {
      const int4 v = *reinterpret_cast<const int4*>(&s.expert[a]);
      const int e4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e4[i] == mine) {
          if (first < 0) first = a + i;
          ++count;
          if (a + i < tid) ++rank;
        }
    }
    const uint32_t lead = __ballot_sync(0xffffffffu, tid < n && first == tid);
    if (lane == 0) s.lead[warp] = lead;
  }
  __syncthreads();
  int groups = 0;
  for (int w = 0; w < kFewChoices / 32; ++w) groups += __popc(s.lead[w]);
  if (tid < n) {
    int at = __popc(s.lead[first >> 5] & ((1u << (first & 31)) - 1));
    for (int w = 0; w < first >> 5; ++w) at += __popc(s.lead[w]);
    s.group_a[at][rank] = tid;
    if (rank == 0) s.group_e[at] = mine, s.group_n[at] = count;
  }
  __syncthreads();
  return groups;
}

template <typename T, int NV>
__global__ void __launch_bounds__(kFewThreads, 1) expert_few_kernel(const ExpertParams p) {
  extern __shared__ __align__(128) uint8_t rings[];
  __shared__ FewShared s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  few_logits<T>(p, s);
  grid_barrier(p, 1);
  const int groups = few_groups<T, NV>(p, s, reinterpret_cast<double*>(rings));  // nothing is copied yet
  const int per1 = p.inter / 8, per2 = (p.hidden + 15) / 16;
  const int units1 = groups * per1, units2 = groups * per2;
  const int warps = gridDim.x * (kFewThreads / 32), me = warp * gridDim.x + blockIdx.x;  // neighbours on other SMs
  const uint32_t ring = smem_u32(rings + warp * kDepth * kChunk);

  Copies<T> w;
  auto open = [&](int second, int u) {
    if (!second && u >= units1) second = 1, u = me;
    w.second = second, w.u = u, w.k = 0;
    w.K = second ? p.inter : p.hidden;
    if (second && u >= units2) return;
    const int group = u / (second ? per2 : per1), row = u - group * (second ? per2 : per1), e = s.group_e[group];
    w.low = second ? static_cast<const T*>(p.down) + ((int64_t)e * p.hidden + row * 16) * p.inter
                   : static_cast<const T*>(p.gate_up) + ((int64_t)e * 2 * p.inter + row * 8) * p.hidden;
    w.high = !second ? (int64_t)p.inter * p.hidden  // past hidden there are no rows of down: the first eight again
             : row * 16 + 8 < p.hidden ? (int64_t)8 * p.inter : 0;
  };
  int put_slot = 0;
  auto copy = [&] {  // one chunk, or an empty group: a row's 512 bytes by each instruction
    if (!(w.second && w.u >= units2)) {
      const int k = w.k + lane * 8;
      const bool there = k < w.K;
      const T* from = w.low + (there ? k : 0);
      const uint32_t to = ring + put_slot * kChunk + (lane >> 3) * 128;
#pragma unroll
      for (int r = 0; r < 8; ++r, from += w.K) {
        const uint32_t at = to + r * kChunkK * 2 + (((lane & 7) ^ r) << 4);
        cp_async_16_or_0(at, from, there);
        cp_async_16_or_0(at + 8 * kChunkK * 2, from + w.high, there);
      }
      w.k += kChunkK;
      if (w.k >= w.K) open(w.second, w.u + warps);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++put_slot == kDepth) put_slot = 0;
  };
  open(0, me);
  for (int i = 0; i < kDepth - 1; ++i) copy();

  // This lane's 16-byte units of rows g and g + 8, and its 16 elements of 64.
  const uint32_t get0 = ring + g * kChunkK * 2 + (((2 * q) ^ g) << 4), get1 = ring + g * kChunkK * 2 + (((2 * q + 1) ^ g) << 4);
  int get_slot = 0;
  float acc[4];
  // acc = rows x this lane's token from col on, K of them, and with `left` their second halves that far
  // behind. Four sums side by side: a product that waits for the last one's sum takes its whole latency.
  auto product = [&](const T* col, int64_t left, int K) {
    float part[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.f;
    for (int c = 0; c < K; c += kChunkK) {
      uint4 b[4][2], rest[4][2];
      auto load = [&](uint4 (&to)[4][2], const T* from) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = c + i * 64 + q * 16;
          to[i][0] = k < K ? *reinterpret_cast<const uint4*>(from + k) : make_uint4(0, 0, 0, 0);
          to[i][1] = k + 8 < K ? *reinterpret_cast<const uint4*>(from + k + 8) : make_uint4(0, 0, 0, 0);
        }
      };
      load(b, col);
      if (left) load(rest, col + left);
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 a[4];  // rows g and g + 8, two units each
        const uint32_t at = get_slot * kChunk + i * 128;
#pragma unroll
        for (int h = 0; h < 4; ++h)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(a[h].x), "=r"(a[h].y), "=r"(a[h].z), "=r"(a[h].w)
                       : "r"((h & 1 ? get1 : get0) + at + (h >> 1) * 8 * kChunkK * 2)
                       : "memory");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a0[4] = {a[h].x, a[2 + h].x, a[h].y, a[2 + h].y};
          const uint32_t a1[4] = {a[h].z, a[2 + h].z, a[h].w, a[2 + h].w};
          mma16816<T>(part[0], a0, b[i][h].x, b[i][h].y);
          mma16816<T>(part[1], a1, b[i][h].z, b[i][h].w);
          if (left) {
            mma16816<T>(part[2], a0, rest[i][h].x, rest[i][h].y);
            mma16816<T>(part[3], a1, rest[i][h].z, rest[i][h].w);
          }
        }
      }
      if (++get_slot == kDepth) get_slot = 0;
      __syncwarp();
      copy();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
  };

  T* act = static_cast<T*>(p.act);
  const int64_t left = (int64_t)p.tokens * p.top_k * p.inter;
  for (int u = me; u < units1; u += warps) {
    const int group = u / per1, row = u - group * per1, n = s.group_n[group];
    // A column past the group's tokens: its first token again.
    product(static_cast<const T*>(p.x) + s.group_a[group][g < n ? g : 0] / p.top_k * p.x_stride, 0, p.hidden);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (2 * q + k < n) {
        const float gate = acc[k], up = acc[2 + k];
        const float v = __fdividef(gate, 1.f + __expf(-gate)) * up;
        T* to = act + (int64_t)s.group_a[group][2 * q + k] * p.inter + row * 8 + g;
        two_halves(v, to[0], to[left]);
      }
  }
  grid_barrier(p, 2);  // the first of down's rows are on their way meanwhile
  for (int u = me; u < units2; u += warps) {
    const int group = u / per2, row = u - group * per2, n = s.group_n[group];
    product(act + (int64_t)s.group_a[group][g < n ? g : 0] * p.inter, left, p.inter);
    const int r = row * 16 + g;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (2 * q + k < n) {
        float* y = p.y + (int64_t)s.group_a[group][2 * q + k] * p.hidden + r;
        y[0] = acc[k];
        if (r + 8 < p.hidden) y[8] = acc[2 + k];
      }
  }
  grid_barrier(p, 3);
  combine<T>(p, s.weight);
  leave(p, &s.last);
}

// ---------------------------------------------------------------- host

struct Layout {
  int64_t logits, sizes, perm, weight, done, xs, act, y, bytes;
  int max_tiles, tile_n, rows1, rows2, stages, slot_b, rows_x, rows_act;
  bool few, direct;
};

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// About how long the tiles of `tile_n` tokens take, in cycles, and the weight rows of an item that take least.
// A stage of 16 KB of weights and its token rows comes at some 52 bytes a cycle from L2 and costs 45 cycles a
// product at least, an item some 2500 besides; items are dealt out in rounds over the SMs. Down's tokens are two
// halves.
struct Tiling {
  double cycles;
  int rows1, rows2;
};
Tiling make_tiling(int64_t tokens, int64_t experts, int top_k, int hidden, int inter, int tile_n, bool direct, int sms) {
  const double rows = (double)tokens * top_k, active = std::min<double>(experts, rows), share = rows / experts;
  // An expert's tokens are its share, more or less: half of those that nearly fill a tile take another.
  const double tiles = direct ? active : active * std::max(1.0, share / tile_n + (share > 0.7 * tile_n ? 0.5 : 0.0));
  auto pick = [&](int64_t n, int k, int columns, int halves, int& best) {
    double least = 1e300;
    for (int r : {128, 64, 32}) {
      const int wide = 128 / r;
      if (tile_n * wide > 272) break;  // at least four stages
      const double stage = std::max({(kSlotA + 128.0 * columns * wide * halves) / 52,
                                     4.0 * wide * halves * std::max(45.0, columns / 2.0), 500.0});
      const double item = 2500 + ((k + kKB - 1) / kKB + wide - 1) / wide * stage;
      const double time = std::ceil(tiles * (double)((n + r - 1) / r) / sms) * item;
      if (time < 0.95 * least) least = time, best = r;
    }
    return least;
  };
  Tiling t = {};
  const int columns = (int)std::min<double>(tile_n, std::max(16.0, share * 1.2));  // of most tiles
  t.cycles = pick(2 * (int64_t)inter, hidden, direct ? tile_n : columns, 1, t.rows1) + pick(hidden, inter, columns, 2, t.rows2);
  return t;
}

// The tiling, from sizes alone, and where each part of the workspace lies.
Layout make_layout(int64_t tokens, int experts, int top_k, int hidden, int inter, int sms) {
  Layout l = {};
  // Few tokens and few weights: the latency of the chain. From some 300 MB of weights on the tcgen05 tiles are
  // faster (7 tokens of 896, 183 MB at most: 37 us, 42 by tiles; 8 of 2048, 604 MB at most: 85 and 82 us).
  l.few = tokens <= kFewTokens && std::min<int64_t>(experts, tokens * top_k) * 6 * hidden * inter <= (300ll << 20);
  l.direct = tokens <= kDirectTokens;
  const int64_t rows = tokens * top_k;
  Tiling best = {1e300, 128, 128};
  if (l.few) {
    l.tile_n = 16;
  } else if (l.direct) {  // a tile per expert
    l.tile_n = (int)up(tokens, 16);
    best = make_tiling(tokens, experts, top_k, hidden, inter, l.tile_n, true, sms);
  } else {
    const double share = (double)rows / experts, most = share + 3 * std::sqrt(share);  // of nearly every expert
    for (int n : {32, 64, 96, 128, 192, 256}) {  // small ones leave the ring more stages
      if (n >= share && n < most && most <= 256) continue;  // some would spill over into a tile of their own
      const Tiling t = make_tiling(tokens, experts, top_k, hidden, inter, n, false, sms);
      if (t.cycles < 0.99 * best.cycles) best = t, l.tile_n = n;  // 2048 tokens of 8 in 64 experts: 256, 320 us, not 192, 345
    }
  }
  l.rows1 = best.rows1, l.rows2 = best.rows2;
  l.max_tiles = (int)(std::min<int64_t>(experts, rows) + (l.direct ? 0 : rows / l.tile_n));
  l.rows_act = l.tile_n <= 64 ? 16 : 32;
  l.rows_x = l.direct ? l.tile_n : l.rows_act;
  // A stage's token rows, of as many chunks as its weights have; for down both halves of them where that leaves
  // four stages (eight up to kDirectTokens tokens, where the stream of weights is what counts), else of those tiles
  // alone that are half full (find_item()). 700 tokens of 3584 through 2 of 16 experts of 2368 take 207 us so, 228
  // with eight; 128 tokens of 2048 through 8 of 64 of 768 127 us, 141 with four.
  const int chunk = (int)up(l.tile_n, l.rows_act) * 128, one = chunk * (128 / l.rows1), two = chunk * (128 / l.rows2);
  l.slot_b = std::max(one, kRing / (kSlotA + 2 * two) >= (l.direct ? 8 : 4) ? 2 * two : two);
  l.stages = std::min(kMaxStages, kRing / (kSlotA + l.slot_b));
  int64_t at = up(sizeof(Header), 256);
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  l.logits = take(tokens * experts * 4);
  l.sizes = take(tokens * experts * 4);
  l.perm = take(tokens * experts * 4);
  l.weight = take(rows * 4);
  l.done = take((std::min<int64_t>(experts, rows) + rows / 32) * 4);  // of the smallest tiles
  l.xs = take(l.direct ? 0 : rows * hidden * 2);
  l.act = take(rows * inter * 4);
  l.y = take(rows * hidden * 4);
  l.bytes = at;
  return l;
}

// Items are counted in 32 bits.
bool items_ok(const Layout& l, int hidden, int inter) {
  const int64_t per = (2 * (int64_t)inter + l.rows1 - 1) / l.rows1 + ((int64_t)hidden + l.rows2 - 1) / l.rows2;
  return l.max_tiles * per <= kMaxItems;
}

bool sizes_ok(int64_t tokens, int experts, int top_k, int hidden, int inter) {
  return tokens >= 0 && experts > 0 && experts <= kMaxExperts && top_k > 0 && top_k <= kMaxTopK && top_k <= experts &&
         hidden > 0 && inter > 0 && hidden % 8 == 0 && inter % 8 == 0 && tokens <= (1 << 24) && hidden <= (1 << 20) &&
         inter <= (1 << 20);
}

template <typename T, int MT>
void launch_router(const ExpertParams& p, int groups, cudaStream_t st) {
  // With more groups than tickets a CTA takes all experts of its group.
  const dim3 grid(groups, groups <= kMaxTickets ? (p.experts + 16 * MT - 1) / (16 * MT) : 1);
  const int threads = MT == 1 ? 512 : 256;
  if (p.experts <= 64) router_kernel<T, MT, 2><<<grid, threads, 0, st>>>(p);
  else if (p.experts <= 128) router_kernel<T, MT, 4><<<grid, threads, 0, st>>>(p);
  else router_kernel<T, MT, 16><<<grid, threads, 0, st>>>(p);
}

template <typename T>
int launch(const CUtensorMap (&maps)[7], const ExpertParams& p, bool few, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_sms());
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  // Cooperative: the CTAs wait for one another's activations, so they must all be resident.
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  // The kernel starts up while the one before it ends.
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = few ? 1 : 2;
  if (few) {
    static SmemAttribute attributes[3];
    const int n = p.experts <= 64 ? 0 : p.experts <= 128 ? 1 : 2;
    auto kernel = n == 0 ? expert_few_kernel<T, 2> : n == 1 ? expert_few_kernel<T, 4> : expert_few_kernel<T, 16>;
    const cudaError_t e = attributes[n].set(reinterpret_cast<const void*>(kernel), kFewSmem);
    if (e != cudaSuccess) return cuda_status(e);
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = kFewSmem;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p));
  }
  const int groups = (p.tokens + kRouterTokens - 1) / kRouterTokens;
  // 16 experts per CTA; 64 for each load of the tokens once those fill the SMs.
  if (groups * (int64_t)((p.experts + 63) / 64) < num_sms() / 2) launch_router<T, 1>(p, groups, st);
  else launch_router<T, 4>(p, groups, st);
  int rc = launch_status();
  if (rc != PKV_OK) return rc;
  if (!p.direct) {
    cudaLaunchConfig_t gather = {};
    gather.gridDim = dim3(8 * num_sms());
    gather.blockDim = dim3(256);
    gather.stream = st;
    gather.attrs = at + 1;
    gather.numAttrs = 1;
    rc = cuda_status(cudaLaunchKernelEx(&gather, gather_kernel, p));
    if (rc != PKV_OK) return rc;
  }
  static SmemAttribute attribute;
  const int smem = 1024 + p.stages * (kSlotA + p.slot_b);
  const cudaError_t e = attribute.set(reinterpret_cast<const void*>(expert_kernel<T>), 1024 + kRing);
  if (e != cudaSuccess) return cuda_status(e);
  cfg.dynamicSmemBytes = smem;
  return cuda_status(cudaLaunchKernelEx(&cfg, expert_kernel<T>, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], maps[6], p));
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_expert_mlp_workspace_bytes(int64_t n_tokens, int32_t num_experts, int32_t top_k, int32_t hidden,
                                                  int32_t intermediate) {
  if (!sizes_ok(n_tokens, num_experts, top_k, hidden, intermediate)) return 0;
  if (!items_ok(make_layout(n_tokens, num_experts, top_k, hidden, intermediate, 148), hidden, intermediate)) return 0;
  // What holds n_tokens holds every smaller call: the layouts change at a few tokens.
  int64_t most = 0;
  for (int64_t t : {(int64_t)1, (int64_t)2, (int64_t)3, (int64_t)4, (int64_t)5, (int64_t)6, (int64_t)7, (int64_t)8, (int64_t)kDirectTokens, n_tokens})
    most = std::max(most, make_layout(std::min(t, n_tokens), num_experts, top_k, hidden, intermediate, 148).bytes);
  return most;
}

extern "C" int pkv_expert_mlp(int32_t dtype, const void* x, int64_t x_stride, int64_t n_tokens, int32_t hidden,
                              int32_t intermediate, int32_t num_experts, int32_t top_k, int32_t renormalize,
                              const void* router, const void* gate_up, const void* down, void* out, int64_t out_stride,
                              void* workspace, int64_t workspace_bytes, int32_t* status_dev, pkv_stream_t stream) {
  if (!router || !gate_up || !down || !workspace) return PKV_ERR_INVALID_ARGUMENT;
  if (n_tokens < 0 || hidden <= 0 || intermediate <= 0 || num_experts <= 0 || top_k <= 0 || top_k > num_experts)
    return PKV_ERR_INVALID_ARGUMENT;
  if (dtype != PKV_F16 && dtype != PKV_BF16) return PKV_ERR_UNSUPPORTED;
  if (!sizes_ok(n_tokens, num_experts, top_k, hidden, intermediate)) return PKV_ERR_UNSUPPORTED;
  if (n_tokens == 0) return PKV_OK;
  if (!x || !out) return PKV_ERR_INVALID_ARGUMENT;
  if (x_stride < hidden || out_stride < hidden || x_stride % 8 || out_stride % 8) return PKV_ERR_INVALID_ARGUMENT;
  auto bits = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  if (((bits(x) | bits(router) | bits(gate_up) | bits(down) | bits(out)) & 15) || (bits(workspace) & 255))
    return PKV_ERR_INVALID_ARGUMENT;
  const Layout l = make_layout(n_tokens, num_experts, top_k, hidden, intermediate, 148);
  if (!items_ok(l, hidden, intermediate)) return PKV_ERR_UNSUPPORTED;
  if (workspace_bytes < l.bytes) return PKV_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ExpertParams p = {};
  p.x = x, p.router = router, p.gate_up = gate_up, p.down = down, p.out = out, p.status = status_dev;
  p.head = reinterpret_cast<Header*>(ws);
  p.logits = reinterpret_cast<float*>(ws + l.logits);
  p.sizes = reinterpret_cast<float*>(ws + l.sizes);
  p.perm = reinterpret_cast<int32_t*>(ws + l.perm);
  p.weight = reinterpret_cast<float*>(ws + l.weight);
  p.done = reinterpret_cast<int32_t*>(ws + l.done);
  p.xs = ws + l.xs;
  p.act = ws + l.act;
  p.y = reinterpret_cast<float*>(ws + l.y);
  p.x_stride = x_stride, p.out_stride = out_stride;
  p.tokens = (int)n_tokens, p.hidden = hidden, p.inter = intermediate, p.experts = num_experts, p.top_k = top_k;
  p.renormalize = renormalize;
  p.max_tiles = l.max_tiles, p.rows1 = l.rows1, p.rows2 = l.rows2;
  p.per1 = (2 * intermediate + l.rows1 - 1) / l.rows1, p.per2 = (hidden + l.rows2 - 1) / l.rows2;
  p.tile_n = l.tile_n;
  p.stages = l.stages, p.slot_b = l.slot_b, p.direct = l.direct, p.rows_x = l.rows_x, p.rows_act = l.rows_act;
  p.drop_y = hidden % 32 == 0 && n_tokens * top_k * hidden * 4 >= kDropBytes;
  p.acc_cols = std::max(l.tile_n, 2 * std::min(l.tile_n, kJointRows));
  p.tmem_cols = 32;
  while (p.tmem_cols < 2u * p.acc_cols) p.tmem_cols *= 2;
  CUtensorMap maps[7];
  int rc = PKV_OK;
  // Token rows: one stack of x, and the values and rests of the activations.
  const uint64_t rows = (uint64_t)n_tokens * top_k;
  auto x_map = [&](CUtensorMap& map, uint32_t box) {
    return l.direct ? make_stack_tensor_map(&map, x, dtype, hidden, n_tokens, 1, box, 1, x_stride)
                    : make_stack_tensor_map(&map, p.xs, dtype, hidden, rows, 1, box, 1);
  };
  auto act_map = [&](CUtensorMap& map, uint32_t box, uint32_t halves) {
    return make_stack_tensor_map(&map, p.act, dtype, intermediate, rows, 2, box, halves);
  };
  if (!l.few) rc = x_map(maps[0], l.rows_x);
  // Operand A of the first product alternates 16 gate rows and their 16 up rows: in one copy where an
  // expert's rows are whole groups of 16, else a copy for each 32.
  p.in16 = intermediate % 16 == 0;
  if (rc == PKV_OK && !l.few)
    rc = p.in16 ? make_split_tensor_map(&maps[1], gate_up, dtype, hidden, intermediate, 2 * (uint64_t)num_experts, 16, 2, l.rows1 / 32)
                : make_stack_tensor_map(&maps[1], gate_up, dtype, hidden, intermediate, 2 * (uint64_t)num_experts, 16, 2);
  if (rc == PKV_OK && !l.few) rc = act_map(maps[2], l.rows_act, 1);
  if (rc == PKV_OK && !l.few) rc = make_stack_tensor_map(&maps[3], down, dtype, intermediate, hidden, num_experts, l.rows2, 1);
  if (!l.few) maps[4] = maps[0], maps[5] = maps[2];
  if (rc == PKV_OK && !l.few && !l.direct && l.rows_act == 32) rc = x_map(maps[4], 128);
  if (rc == PKV_OK && !l.few && l.rows_act == 32) rc = act_map(maps[5], 128, 1);
  if (rc == PKV_OK && !l.few) rc = act_map(maps[6], l.rows_act, 2);
  if (rc != PKV_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == PKV_F16 ? launch<__half>(maps, p, l.few, st) : launch<__nv_bfloat16>(maps, p, l.few, st);
}
