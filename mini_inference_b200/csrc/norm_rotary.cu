// Rotary positions of decoder layers that normalise each query and key head first, with
// positions on several axes, fused with the KV append; and those positions, from the images and
// video in a prompt.
//
// A head x of d elements becomes y = x / sqrt(mean(x^2) + eps) * w, and its pair i is then turned
// by the angle positions[axes[i]] * inv_freq[i]:
//   (a, b) -> (a cos - b sin, b cos + a sin) * attention_factor
// with a, b the elements (2i, 2i + 1) or (i, i + rotary / 2). Angles are reduced to a fraction of
// a turn in float64 (a float32 angle at position 2^20 is off by up to 2^-4 radians); the sum of
// squares, the norm and the rotation are float32, and each element is rounded to the storage type
// once, where a norm kernel and a rotation kernel would round twice.
//
// No counterpart in the reference, whose layers neither normalise heads nor have more than one
// axis (engine/model.py:190-251).
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace pkv {
namespace {

constexpr int kMaxHalf = 256;  // pairs of a head
constexpr int kMaxAxes = 4;
constexpr int kThreads = 256;  // at most

struct NormRotaryParams {
  const void* qkv;
  const int64_t* positions;
  const int32_t* axes;
  const double* inv_freq;
  const void* q_weight;
  const void* k_weight;
  void* q_out;
  void* k_out;
  void* v_out;
  void* k_pool;
  void* v_pool;
  const int64_t* slots;
  int32_t* status;
  int64_t pos_stride, qkv_stride, q_st, q_sh, k_st, k_sh, v_st, v_sh, layer_base;
  float factor, eps;
  int hq, hkv, d, half, bs, nbt, num_axes;
  int lanes_log2;  // lanes of a head: the power of two that holds its units
  int v_log2;      // units of a V head, rounded up to a power of two
};

template <typename T, int EW> struct alignas(EW * sizeof(T)) Vec {
  T v[EW];
};

// A token's slot, or -1: none.
__device__ __forceinline__ int64_t token_slot(const NormRotaryParams& p, int64_t t) {
  const int64_t slot = p.slots ? p.slots[t] : -1;
  if (slot < (int64_t)p.nbt * p.bs) return slot;
  report(p.status, PKV_ERR_OUT_OF_RANGE);
  return -1;
}

// Cos and sin of a token's pair i, times the factor.
__device__ __forceinline__ float2 pair_angle(const NormRotaryParams& p, int64_t t, int i) {
  int axis = p.axes ? p.axes[i] : 0;
  if ((unsigned)axis >= (unsigned)p.num_axes) {
    report(p.status, PKV_ERR_OUT_OF_RANGE);
    axis = 0;
  }
  const int64_t pos = p.positions[axis * p.pos_stride + t];
  if (pos < 0) report(p.status, PKV_ERR_OUT_OF_RANGE);
  const double turns = (double)pos * p.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
  const float r = (float)(turns - rint(turns));                             // [-1/2, 1/2]
  float s, c;
  sincospif(2.f * r, &s, &c);
  return make_float2(c * p.factor, s * p.factor);
}

// One CTA per token. A head is held by a group of 2 to 32 lanes: a lane's unit is 16 elements a[8] and
// b[8], pairs that rotate together (half a rotation apart, or side by side), or past the rotated
// part two vectors that do not. The group sums the squares by shuffles, so a head is read once and
// written once. Norm weight, cos, sin and factor are multiplied once per token and pair, into four
// numbers for q and four for k:
//   a' = (a A - b B) rs,  b' = (b C + a D) rs,  A = wa cos, B = wb sin, C = wb cos, D = wa sin
// (A = wa, C = wb, no b in a' and no a in b' past the rotated part), so that a head costs three products an element
// and no weights: the kernel is bound by instructions as much as by bytes. 8192 tokens of 28 / 4 heads
// of 128 (bf16, three axes, appended) take 30 us = 5.0 TB/s, 0.77 of the copy bandwidth; with weights,
// cos and sin applied one after another they took 45, with each head's load in its own turn 33. Two
// elements at a time by paired fp32 instructions. Four tokens per CTA with their loads ahead of the
// angles were slower (61-120 us).
// REST: there is a part that is not rotated (its selects cost a whole-head rotation 5 %: 31.6 us).
template <typename T, bool INTER, bool NORM, bool REST>
__global__ void __launch_bounds__(kThreads) norm_rotary_kernel(const NormRotaryParams p) {
  __shared__ float4 table[NORM ? 2 : 1][8][32];  // q and k: {A A B B}, {C C D D} of two pairs, by unit
  using V = Vec<T, 8>;
  const int64_t t = blockIdx.x;
  const int heads = p.hq + p.hkv;
  const T* row = static_cast<const T*>(p.qkv) + t * p.qkv_stride;
  const int rot_units = p.half / 8, rest = p.d - 2 * p.half;
  const int64_t slot = token_slot(p, t);
  // The elements of unit u's pair e.
  auto first = [&](int u, int e) { return u < rot_units ? INTER ? 16 * u + 2 * e : 8 * u + e : 2 * p.half + 16 * (u - rot_units) + e; };
  auto second = [&](int u, int e) { return first(u, e) + (u < rot_units ? INTER ? 1 : p.half : 8); };
  const int units = rot_units + (rest + 15) / 16;
  const int lanes = 1 << p.lanes_log2, sub = threadIdx.x & (lanes - 1);
  const int groups = blockDim.x >> p.lanes_log2;
  const bool has_a = sub < units;
  const int ca = first(sub, 0);
  const int cb = INTER && sub < rot_units ? ca + 8 : second(sub, 0);
  const bool has_b = has_a && cb < p.d;
  // A group's next head is loaded ahead, the first before the angles.
  uint4 next_a = make_uint4(0, 0, 0, 0), next_b = next_a;
  auto load = [&](int head) {
    if (has_a && head < heads) next_a = *reinterpret_cast<const uint4*>(row + head * p.d + ca);
    if (has_b && head < heads) next_b = *reinterpret_cast<const uint4*>(row + head * p.d + cb);
  };
  load(threadIdx.x >> p.lanes_log2);
  for (int i = threadIdx.x; i < 8 * units; i += blockDim.x) {
    const int u = i >> 3, e = i & 7;
    const float2 cs = u < rot_units ? pair_angle(p, t, i) : make_float2(1.f, 0.f);
#pragma unroll
    for (int k = 0; k < (NORM ? 2 : 1); ++k) {
      float wa = 1.f, wb = 1.f;
      if (NORM) {
        const T* w = static_cast<const T*>(k ? p.k_weight : p.q_weight);
        const int cb = second(u, e);
        wa = Dt<T>::to_f(w[first(u, e)]);
        wb = cb < p.d ? Dt<T>::to_f(w[cb]) : 0.f;
      }
      float* ab = reinterpret_cast<float*>(&table[k][e & 6][u]) + (e & 1);
      float* cd = reinterpret_cast<float*>(&table[k][e | 1][u]) + (e & 1);
      ab[0] = wa * cs.x, ab[2] = wb * cs.y;
      cd[0] = wb * cs.x, cd[2] = wa * cs.y;
    }
  }
  __syncthreads();
  const int64_t in_block = slot >= 0 ? ((p.layer_base + slot / p.bs) * p.hkv * p.bs + slot % p.bs) * p.d : 0;
  const int64_t head_step = (int64_t)p.bs * p.d;

  for (int h0 = 0; h0 < heads; h0 += groups) {  // the same count for every lane: the shuffles need them all
    const int head = h0 + (threadIdx.x >> p.lanes_log2);
    const bool on_a = has_a && head < heads, on_b = has_b && head < heads;
    const uint4 va = next_a, vb = next_b;
    load(head + groups);
    const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
    float2 a[4], b[4];  // pairs 2 j and 2 j + 1
    const bool side = INTER && sub < rot_units;  // pair e is word e of the two vectors
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = Dt<T>::unpack(INTER && side ? (j < 2 ? wa[(2 * j) & 3] : wb[(2 * j) & 3]) : wa[j]);
      const float2 y = Dt<T>::unpack(INTER && side ? (j < 2 ? wa[(2 * j + 1) & 3] : wb[(2 * j + 1) & 3]) : wb[j]);
      a[j] = INTER && side ? make_float2(x.x, y.x) : x;
      b[j] = INTER && side ? make_float2(x.y, y.y) : y;
    }
    float rs = 1.f;
    if constexpr (NORM) {
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = ffma2(b[j], b[j], ffma2(a[j], a[j], ss));
      float sum = ss.x + ss.y;
      for (int o = lanes >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      rs = rsqrtf(sum / (float)p.d + p.eps);
    }
    if (!on_a) continue;  // the group's own lanes only: shuffles are above
    const float2 rs2 = make_float2(rs, rs);
    const int which = NORM && head >= p.hq ? 1 : 0;
    uint32_t oa[4], ob[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 ab = table[which][2 * j][sub], cd = table[which][2 * j + 1][sub];
      // Past the rotated part there is no pair: an infinity times nothing would be the other's NaN (-0 to add, which
      // keeps a -0). Asked of `rest` too, which REST implies: 54 registers, 78 without, where six CTAs fit an SM in
      // place of seven (1013 rows of half-rotated heads 6.1 and 7.4 us).
      float2 cross_a = a[j], cross_b = b[j];
      if (REST && rest && sub >= rot_units) cross_a = make_float2(-0.f, -0.f), cross_b = make_float2(0.f, 0.f);
      float2 x = ffma2(a[j], make_float2(ab.x, ab.y), fmul2(make_float2(-cross_b.x, -cross_b.y), make_float2(ab.z, ab.w)));
      float2 y = INTER ? ffma2(cross_a, make_float2(cd.z, cd.w), fmul2(b[j], make_float2(cd.x, cd.y)))
                       : ffma2(b[j], make_float2(cd.x, cd.y), fmul2(cross_a, make_float2(cd.z, cd.w)));
      if (NORM) x = fmul2(x, rs2), y = fmul2(y, rs2);
      if (INTER && side) {
        (j < 2 ? oa : ob)[(2 * j) & 3] = Dt<T>::pack(x.x, y.x);
        (j < 2 ? oa : ob)[(2 * j + 1) & 3] = Dt<T>::pack(x.y, y.y);
      } else {
        oa[j] = Dt<T>::pack(x.x, x.y);
        ob[j] = Dt<T>::pack(y.x, y.y);
      }
    }
    auto put = [&](T* base) {
      *reinterpret_cast<uint4*>(base + ca) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
      if (on_b) *reinterpret_cast<uint4*>(base + cb) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
    };
    if (head < p.hq) {
      put(static_cast<T*>(p.q_out) + t * p.q_st + head * p.q_sh);
    } else {
      const int kh = head - p.hq;
      if (p.k_out) put(static_cast<T*>(p.k_out) + t * p.k_st + kh * p.k_sh);
      if (slot >= 0) put(static_cast<T*>(p.k_pool) + in_block + kh * head_step);
    }
  }
  if (p.v_out || slot >= 0) {
    for (int u = threadIdx.x; u < p.hkv << p.v_log2; u += blockDim.x) {
      const int kh = u >> p.v_log2, c = (u & ((1 << p.v_log2) - 1)) * 8;
      if (c >= p.d) continue;
      const V x = *reinterpret_cast<const V*>(row + (heads + kh) * p.d + c);
      if (p.v_out) *reinterpret_cast<V*>(static_cast<T*>(p.v_out) + t * p.v_st + kh * p.v_sh + c) = x;
      if (slot >= 0) *reinterpret_cast<V*>(static_cast<T*>(p.v_pool) + in_block + kh * head_step + c) = x;
    }
  }
}

// Rows, heads or halves that do not start on 16 bytes: a warp per head, an element at a time. The
// head is read twice (its squares, then its elements), the second time from L1. 8192 tokens of 28 / 4 heads of
// 72 (bf16, three axes, appended) take 98 us = 0.86 TB/s, one token 6.9: bound by its instructions, two bytes a lane.
template <typename T, bool INTER, bool NORM>
__global__ void __launch_bounds__(kThreads) norm_rotary_any_kernel(const NormRotaryParams p) {
  __shared__ float2 cs[kMaxHalf];
  const int64_t t = blockIdx.x;
  const int64_t slot = token_slot(p, t);
  for (int i = threadIdx.x; i < p.half; i += blockDim.x) cs[i] = pair_angle(p, t, i);
  __syncthreads();
  const T* row = static_cast<const T*>(p.qkv) + t * p.qkv_stride;
  const int heads = p.hq + p.hkv, lane = threadIdx.x & 31;
  const int64_t in_block = slot >= 0 ? ((p.layer_base + slot / p.bs) * p.hkv * p.bs + slot % p.bs) * p.d : 0;
  const int64_t head_step = (int64_t)p.bs * p.d;
  for (int head = threadIdx.x >> 5; head < heads + p.hkv; head += blockDim.x >> 5) {
    const T* x = row + head * p.d;
    const bool is_v = head >= heads;
    float rs = 1.f;
    const T* w = nullptr;
    if (NORM && !is_v) {
      float ss = 0.f;
      for (int c = lane; c < p.d; c += 32) {
        const float f = Dt<T>::to_f(x[c]);
        ss += f * f;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rs = rsqrtf(ss / (float)p.d + p.eps);
      w = static_cast<const T*>(head < p.hq ? p.q_weight : p.k_weight);
    }
    T *one, *two = nullptr;  // where the head goes
    const int kh = head - (is_v ? heads : p.hq);
    if (head < p.hq) {
      one = static_cast<T*>(p.q_out) + t * p.q_st + head * p.q_sh;
    } else {
      T* out = static_cast<T*>(is_v ? p.v_out : p.k_out);
      one = out ? out + t * (is_v ? p.v_st : p.k_st) + kh * (is_v ? p.v_sh : p.k_sh) : nullptr;
      if (slot >= 0) two = static_cast<T*>(is_v ? p.v_pool : p.k_pool) + in_block + kh * head_step;
    }
    auto put = [&](int c, T y) {
      if (one) one[c] = y;
      if (two) two[c] = y;
    };
    auto get = [&](int c) { return Dt<T>::to_f(x[c]) * (w ? rs * Dt<T>::to_f(w[c]) : 1.f); };
    const int pairs = is_v ? 0 : p.half;
    for (int i = lane; i < pairs; i += 32) {
      const int ca = INTER ? 2 * i : i, cb = INTER ? 2 * i + 1 : i + p.half;
      const float a = get(ca), b = get(cb);
      const float2 cw = cs[i];
      put(ca, Dt<T>::from_f(a * cw.x - b * cw.y));
      put(cb, Dt<T>::from_f(b * cw.x + a * cw.y));
    }
    for (int c = 2 * pairs + lane; c < p.d; c += 32) put(c, w ? Dt<T>::from_f(get(c)) : x[c]);
  }
}

int log2_up(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

template <typename T>
int launch(NormRotaryParams p, int64_t n, bool vec16, bool inter, cudaStream_t st) {
  const bool norm = p.q_weight != nullptr;
  const int units = p.half / 8 + (p.d - 2 * p.half + 15) / 16;
  p.lanes_log2 = std::max(1, log2_up(units));
  p.v_log2 = log2_up(p.d / 8);
  if (!vec16 || units > 32) {
    const int warps = std::min(kThreads / 32, p.hq + 2 * p.hkv);
    auto kernel = norm ? inter ? norm_rotary_any_kernel<T, true, true> : norm_rotary_any_kernel<T, false, true>
                       : inter ? norm_rotary_any_kernel<T, true, false> : norm_rotary_any_kernel<T, false, false>;
    kernel<<<(unsigned)n, warps * 32, 0, st>>>(p);
    return launch_status();
  }
  const int work = ((p.hq + p.hkv) << p.lanes_log2) + (p.v_out || p.slots ? p.hkv << p.v_log2 : 0);
  // Few tokens: a unit per thread, for latency. More than the SMs hold at once: several units per thread,
  // so that more tokens are under way. 28 / 4 heads of 128, one, three and five units per thread:
  // 8192 tokens 45, 33 and 30 us; 1013 tokens of 32 / 8 heads 8.0, 6.0 and 6.5 us.
  const int per = n > 16 * num_sms() ? 5 : n > 4 * num_sms() ? 3 : 1;
  const int threads = std::min(kThreads, std::max(64, (work + per * 32 - 1) / (per * 32) * 32));
  auto pick = [&](auto rest) {
    constexpr bool R = decltype(rest)::value;
    return norm ? inter ? norm_rotary_kernel<T, true, true, R> : norm_rotary_kernel<T, false, true, R>
                : inter ? norm_rotary_kernel<T, true, false, R> : norm_rotary_kernel<T, false, false, R>;
  };
  auto kernel = 2 * p.half < p.d ? pick(std::true_type{}) : pick(std::false_type{});
  kernel<<<(unsigned)n, threads, 0, st>>>(p);
  return launch_status();
}

struct MediaParams {
  const int64_t* positions;
  const int32_t* cu;
  const int32_t* seq_rows;
  const int32_t* media;
  const int32_t* counts;
  int64_t* out;
  int32_t* status;
  int64_t n, out_stride;
  int num_seqs, rows, max_spans;
};

constexpr int kStaged = 1024;  // sequences whose starts fit the CTA's shared memory

// A thread per token: its sequence by bisection, then its sequence's spans one after another up to the
// token (a warp's tokens mostly read the same ones). 32 bytes a token; bound by the chain of loads, so
// the sequences' starts come in one round, a thread's first four spans with their count, and each
// further four before the last are worked on (one after another by dependent loads: 64
// sequences of one token 3.9 us captured, now 3.4; 32 K packed tokens of up to 12 spans 5.1, now 4.9).
__global__ void __launch_bounds__(kThreads) media_positions_kernel(const MediaParams p) {
  __shared__ int32_t starts[kStaged + 1];
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const bool token = t < p.n;
  const int64_t at = token ? p.positions[t] : 0;
  int seq = (int)t;
  if (p.cu) {
    const int32_t* cu = p.cu;
    if (p.num_seqs <= kStaged) {
      for (int i = threadIdx.x; i <= p.num_seqs; i += blockDim.x) starts[i] = p.cu[i];
      __syncthreads();
      cu = starts;
    }
    int lo = 0, hi = p.num_seqs;  // the last sequence that starts at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    if (lo >= p.num_seqs || t < cu[lo]) return;
    seq = lo;
  }
  if (!token) return;
  const int row = p.seq_rows ? p.seq_rows[seq] : seq;
  if (row >= p.rows) report(p.status, PKV_ERR_OUT_OF_RANGE);
  const bool any = row >= 0 && row < p.rows && p.max_spans > 0;
  const int32_t* m = p.media + (any ? (int64_t)row * p.max_spans * 5 : 0);
  int32_t next[4][5];
  auto fetch = [&](int j0) {  // spans j0 .. j0 + 3, within the row
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 5; ++k) next[j][k] = j0 + j < p.max_spans ? m[(j0 + j) * 5 + k] : 0;
  };
  int spans = 0;
  if (any) {
    spans = p.counts[row];
    fetch(0);
    if (spans < 0 || spans > p.max_spans) {
      report(p.status, PKV_ERR_OUT_OF_RANGE);
      spans = 0;
    }
  } else if (row >= 0 && row < p.rows && p.counts[row] != 0) {
    report(p.status, PKV_ERR_OUT_OF_RANGE);
  }
  int64_t lag = 0, end = 0;  // how far positions are behind indexes; the last span's end
  int64_t x0 = at, x1 = at, x2 = at;
  bool inside = false, more = true;
  for (int j0 = 0; j0 < spans && more; j0 += 4) {
    int32_t now[4][5];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 5; ++k) now[j][k] = next[j][k];
    if (j0 + 4 < spans) fetch(j0 + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!more || j0 + j >= spans) continue;
      const int64_t start = now[j][0], frames = now[j][1], height = now[j][2], width = now[j][3], step = now[j][4];
      if (start < end || frames < 1 || height < 1 || width < 1 || step < 0) {
        report(p.status, PKV_ERR_OUT_OF_RANGE);
        more = false;
        continue;
      }
      if (start > at) {
        more = false;
        continue;
      }
      const int64_t plane = height * width, r = at - start;
      // In 64 bits only planes and spans past 32: a division of 64 bits is some hundred instructions.
      const bool small = plane <= 0x7fffffff;
      const int64_t size = small ? frames * plane : r / plane < frames ? r + 1 : frames * plane;  // past r is enough
      if (r < size) {
        int64_t f, y, x;
        if (small && size <= 0xffffffffll) {
          const uint32_t in = (uint32_t)r % (uint32_t)plane;
          f = (uint32_t)r / (uint32_t)plane, y = in / (uint32_t)width, x = in % (uint32_t)width;
        } else {
          const int64_t in = r % plane;
          f = r / plane, y = in / width, x = in % width;
        }
        x0 = start - lag + f * step, x1 = start - lag + y, x2 = start - lag + x;
        inside = true, more = false;
        continue;
      }
      end = start + size;
      lag += size - max(max((frames - 1) * step + 1, height), width);
    }
  }
  if (!inside) x0 = x1 = x2 = at - lag;
  p.out[t] = x0;
  p.out[p.out_stride + t] = x1;
  p.out[2 * p.out_stride + t] = x2;
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_norm_rotary_append(const pkv_pool* pool, int32_t layer, const void* qkv, int64_t qkv_stride,
                                      int64_t n_tokens, int32_t num_q_heads, const int64_t* positions,
                                      int64_t positions_stride, const int32_t* axes, int32_t num_axes,
                                      const double* inv_freq, int32_t rotary_dim, int32_t interleaved,
                                      float attention_factor, const void* q_weight, const void* k_weight, float eps,
                                      void* q_out, int64_t q_out_stride_t, int64_t q_out_stride_h, void* k_out,
                                      int64_t k_out_stride_t, int64_t k_out_stride_h, void* v_out,
                                      int64_t v_out_stride_t, int64_t v_out_stride_h, const int64_t* slot_mapping,
                                      int32_t* status_dev, pkv_stream_t stream) {
  if (!pool || n_tokens < 0 || n_tokens > 0x7fffffff || num_q_heads <= 0) return PKV_ERR_INVALID_ARGUMENT;
  const int d = pool->head_dim, hkv = pool->num_kv_heads;
  if (d <= 0 || hkv <= 0 || num_q_heads % hkv || rotary_dim <= 0 || rotary_dim > d || rotary_dim % 2 ||
      (interleaved != 0 && interleaved != 1))
    return PKV_ERR_INVALID_ARGUMENT;
  if (num_axes < 1 || num_axes > kMaxAxes || (num_axes > 1 && positions_stride < n_tokens) || (num_axes > 1 && !axes))
    return PKV_ERR_INVALID_ARGUMENT;
  if ((q_weight == nullptr) != (k_weight == nullptr) || !(eps >= 0.f)) return PKV_ERR_INVALID_ARGUMENT;
  if (slot_mapping && (layer < 0 || layer >= pool->num_layers || !pool->k || !pool->v || pool->block_size <= 0 ||
                       pool->num_blocks_total <= 0))
    return PKV_ERR_INVALID_ARGUMENT;
  if ((pool->dtype != PKV_F16 && pool->dtype != PKV_BF16) || rotary_dim / 2 > kMaxHalf) return PKV_ERR_UNSUPPORTED;
  const int64_t row = ((int64_t)num_q_heads + 2 * (int64_t)hkv) * d;
  if (qkv_stride < row) return PKV_ERR_INVALID_ARGUMENT;
  if (row > (1 << 30)) return PKV_ERR_UNSUPPORTED;  // a row's elements are counted in 32 bits
  if (n_tokens == 0) return PKV_OK;
  if (!qkv || !positions || !inv_freq || !q_out) return PKV_ERR_INVALID_ARGUMENT;
  if (!slot_mapping && !k_out) return PKV_ERR_INVALID_ARGUMENT;  // the rotated keys must go somewhere
  NormRotaryParams p = {};
  p.qkv = qkv, p.positions = positions, p.axes = axes, p.inv_freq = inv_freq;
  p.q_weight = q_weight, p.k_weight = k_weight;
  p.q_out = q_out, p.k_out = k_out, p.v_out = v_out;
  p.k_pool = pool->k, p.v_pool = pool->v, p.slots = slot_mapping, p.status = status_dev;
  p.pos_stride = num_axes > 1 ? positions_stride : 0;
  p.qkv_stride = qkv_stride;
  p.q_st = q_out_stride_t, p.q_sh = q_out_stride_h;
  p.k_st = k_out ? k_out_stride_t : 0, p.k_sh = k_out ? k_out_stride_h : 0;
  p.v_st = v_out ? v_out_stride_t : 0, p.v_sh = v_out ? v_out_stride_h : 0;
  p.layer_base = slot_mapping ? (int64_t)layer * pool->num_blocks_total : 0;
  p.factor = attention_factor, p.eps = eps;
  p.hq = num_q_heads, p.hkv = hkv, p.d = d, p.half = rotary_dim / 2;
  p.bs = pool->block_size, p.nbt = pool->num_blocks_total, p.num_axes = num_axes;
  auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
  const uintptr_t rows = bits(qkv) | bits(q_out) | bits(k_out) | bits(v_out) | bits(q_weight) | bits(k_weight) |
                         (slot_mapping ? bits(pool->k) | bits(pool->v) : 0);
  if ((rows & 1) || (bits(inv_freq) & 7) || (bits(positions) & 7) || (bits(slot_mapping) & 7) || (bits(axes) & 3))
    return PKV_ERR_INVALID_ARGUMENT;
  // 16-byte accesses where every row, head and half starts on 16 bytes; else one element at a time.
  const int64_t parts = qkv_stride | p.q_st | p.q_sh | p.k_st | p.k_sh | p.v_st | p.v_sh | d | p.half;
  const bool vec16 = (rows & 15) == 0 && (parts & 7) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return pool->dtype == PKV_F16 ? launch<__half>(p, n_tokens, vec16, interleaved != 0, st)
                                : launch<__nv_bfloat16>(p, n_tokens, vec16, interleaved != 0, st);
}

extern "C" int pkv_media_positions(const int64_t* positions, int64_t n_tokens, const int32_t* cu_seqlens,
                                   int32_t num_seqs, const int32_t* seq_rows, const int32_t* media,
                                   const int32_t* media_counts, int32_t rows, int32_t max_spans, int64_t* out,
                                   int64_t out_stride, int32_t* status_dev, pkv_stream_t stream) {
  if (n_tokens < 0 || n_tokens > 0x7fffffff || num_seqs < 0 || rows < 0 || max_spans < 0) return PKV_ERR_INVALID_ARGUMENT;
  if (max_spans > 0x7fffffff / 5 - 4) return PKV_ERR_UNSUPPORTED;  // a row's numbers are counted in 32 bits
  if (!cu_seqlens && n_tokens != num_seqs) return PKV_ERR_INVALID_ARGUMENT;
  if (n_tokens == 0) return PKV_OK;
  if (!positions || !out || out_stride < n_tokens) return PKV_ERR_INVALID_ARGUMENT;
  if (!media_counts && rows > 0) return PKV_ERR_INVALID_ARGUMENT;
  if (!media && rows > 0 && max_spans > 0) return PKV_ERR_INVALID_ARGUMENT;
  auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
  if (((bits(positions) | bits(out)) & 7) || ((bits(cu_seqlens) | bits(seq_rows) | bits(media) | bits(media_counts)) & 3))
    return PKV_ERR_INVALID_ARGUMENT;
  MediaParams p = {positions, cu_seqlens, seq_rows, media, media_counts, out, status_dev, n_tokens, out_stride,
                   num_seqs, rows, max_spans};
  const int threads = n_tokens >= kThreads * num_sms() ? kThreads : 128;
  media_positions_kernel<<<(unsigned)((n_tokens + threads - 1) / threads), threads, 0,
                           reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}
