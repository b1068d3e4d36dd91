// Rotary positions in the layouts pkv_rope_append does not take: pairs side by side
// (interleaved) or half a rotation apart, over the first part of each head only, with
// frequencies of the caller's choosing (scaled for long contexts), fused with the KV append.
//
// For pair i of a head at position p, angle a = p * inv_freq[i]:
//   (x, y) -> (x cos a - y sin a, y cos a + x sin a) * attention_factor
// with x, y the elements (2i, 2i + 1) or (i, i + rotary / 2). The angle is
// reduced to a fraction of a turn in float64: a float32 angle at position 2^20 is off by up
// to 2^-4 radians. No table of positions has to be built or read. cos and sin, the
// products and the sums are float32; each element is rounded to the storage type once.
//
// No counterpart in the reference, whose RotaryEmbedding rotates whole heads in halves at
// unscaled frequencies (engine/model.py:190-224).
#include <algorithm>

#include "common.cuh"

namespace pkv {
namespace {

constexpr int kMaxHalf = 256;  // pairs of a head: head_dim <= 512
constexpr int kThreads = 256;   // at most

// n / d for n d < 2^32 by a multiplication with ceil(2^32 / d), whose excess over 2^32 / d is
// below one: n times it stays below 2^32 / d.
struct Quotient {
  uint32_t d = 1, m = 0;
  Quotient() = default;
  explicit Quotient(uint32_t x) : d(x), m(x > 1 ? (uint32_t)(((1ull << 32) + x - 1) / x) : 0) {}
  __device__ int operator()(int n) const { return d > 1 ? (int)__umulhi((uint32_t)n, m) : n; }
};

struct RotaryParams {
  const void* qkv;
  const int64_t* positions;
  const double* inv_freq;
  void* q_out;
  void* k_out;
  void* v_out;
  void* k_pool;
  void* v_pool;
  const int64_t* slots;
  int32_t* status;
  int64_t qkv_stride, q_st, q_sh, k_st, k_sh, v_st, v_sh, layer_base;
  float factor;
  int32_t hq, hkv, d, half, bs, nbt;
  Quotient per_head, per_rest, per_v;  // a head's units: rotated, copied, of V
};

template <typename T, int EW> struct alignas(EW * sizeof(T)) Vec {
  T v[EW];
};

// One CTA per token: the pairs' cos and sin once into shared memory, then every head's
// units from there. Bound by the rows' bytes, or by the chain position, angles, barrier, rows
// when tokens are few: 8192 tokens of 28 / 4 heads of 128 (bf16, appended as they are rotated)
// take 29.8 us = 5.1 TB/s, 0.78 of the copy bandwidth; 64 tokens 2.8 us. Several tokens per
// CTA or the next unit's loads ahead of this one's stores were slower (43-53 us), and so were the
// first unit's loads ahead of the angles (33 us). A unit is EW pairs: two vectors of EW elements, half a rotation apart
// or side by side; the elements past the rotated part and the V rows are copied.
template <typename T, int EW, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  __shared__ float2 cs[kMaxHalf];
  using V = Vec<T, EW>;
  const int64_t t = blockIdx.x;
  const int64_t pos = p.positions[t];
  int64_t slot = p.slots ? p.slots[t] : -1;
  if (slot >= (int64_t)p.nbt * p.bs) {
    if (threadIdx.x == 0) report(p.status, PKV_ERR_OUT_OF_RANGE);
    slot = -1;
  }
  if (pos < 0 && threadIdx.x == 0) report(p.status, PKV_ERR_OUT_OF_RANGE);
  for (int i = threadIdx.x; i < p.half; i += blockDim.x) {
    const double turns = (double)pos * p.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
    const float r = (float)(turns - rint(turns));                             // [-1/2, 1/2]
    float s, c;
    sincospif(2.f * r, &s, &c);
    cs[i] = make_float2(c * p.factor, s * p.factor);
  }
  __syncthreads();
  const T* row = static_cast<const T*>(p.qkv) + t * p.qkv_stride;
  const int heads = p.hq + p.hkv, per_head = p.half / EW;
  const int rest = (p.d - 2 * p.half) / EW, per_v = p.d / EW;
  const int rot_units = heads * per_head, rest_units = heads * rest;
  const bool want_v = p.v_out || slot >= 0;
  const int units = rot_units + rest_units + (want_v ? p.hkv * per_v : 0);
  const int64_t in_block = slot >= 0 ? ((p.layer_base + slot / p.bs) * p.hkv * p.bs + slot % p.bs) * p.d : 0;
  const int64_t head_step = (int64_t)p.bs * p.d;
  auto put = [&](int head, int c, const V& x) {  // element c of a q or k head
    if (head < p.hq) {
      *reinterpret_cast<V*>(static_cast<T*>(p.q_out) + t * p.q_st + head * p.q_sh + c) = x;
    } else {
      const int kh = head - p.hq;
      if (p.k_out) *reinterpret_cast<V*>(static_cast<T*>(p.k_out) + t * p.k_st + kh * p.k_sh + c) = x;
      if (slot >= 0) *reinterpret_cast<V*>(static_cast<T*>(p.k_pool) + in_block + kh * head_step + c) = x;
    }
  };
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    if (u < rot_units) {
      const int head = p.per_head(u), i0 = (u - head * per_head) * EW;  // first pair
      const int ca = INTER ? 2 * i0 : i0, cb = INTER ? 2 * i0 + EW : i0 + p.half;
      V a = *reinterpret_cast<const V*>(row + head * p.d + ca);
      V b = *reinterpret_cast<const V*>(row + head * p.d + cb);
#pragma unroll
      for (int e = 0; e < EW; ++e) {
        // INTER: the two vectors hold pairs (a0 a1) (a2 a3) .. (b0 b1) ..; pair e of the unit.
        T& x = INTER ? (2 * e < EW ? a.v[(2 * e) % EW] : b.v[(2 * e) % EW]) : a.v[e];
        T& y = INTER ? (2 * e + 1 < EW ? a.v[(2 * e + 1) % EW] : b.v[(2 * e + 1) % EW]) : b.v[e];
        const float2 w = cs[i0 + e];
        const float fx = Dt<T>::to_f(x), fy = Dt<T>::to_f(y);
        x = Dt<T>::from_f(fx * w.x - fy * w.y);
        y = Dt<T>::from_f(fy * w.x + fx * w.y);
      }
      put(head, ca, a);
      put(head, cb, b);
    } else if (u < rot_units + rest_units) {
      const int w = u - rot_units, head = p.per_rest(w), c = 2 * p.half + (w - head * rest) * EW;
      put(head, c, *reinterpret_cast<const V*>(row + head * p.d + c));
    } else {
      const int w = u - rot_units - rest_units, kh = p.per_v(w), c = (w - kh * per_v) * EW;
      const V x = *reinterpret_cast<const V*>(row + (heads + kh) * p.d + c);
      if (p.v_out) *reinterpret_cast<V*>(static_cast<T*>(p.v_out) + t * p.v_st + kh * p.v_sh + c) = x;
      if (slot >= 0) *reinterpret_cast<V*>(static_cast<T*>(p.v_pool) + in_block + kh * head_step + c) = x;
    }
  }
}

template <typename T>
int launch(RotaryParams p, int64_t n, bool vec16, bool inter, cudaStream_t st) {
  // Few tokens: a unit per thread, for latency. More than the SMs hold at once: four units
  // per thread, so that more tokens are under way (a CTA's chain is position, angles, rows).
  // 28 / 4 heads of 128, one and four units: 64 tokens 2.8 and 3.4 us, 592 tokens 4.0 and 4.2, 900
  // tokens 5.8 and 5.1, 8192 tokens 36 and 30.
  const int ew = vec16 ? 8 : 1;
  p.per_head = Quotient(p.half / ew);
  p.per_rest = Quotient(std::max(1, (p.d - 2 * p.half) / ew));
  p.per_v = Quotient(p.d / ew);
  const int units = (p.hq + p.hkv) * (p.d - p.half) / ew + (p.v_out || p.slots ? p.hkv * p.d / ew : 0);
  const int per = n > 4 * num_sms() ? 4 : 1;
  const int threads = std::min(kThreads, std::max(64, (units + per * 32 - 1) / (per * 32) * 32));
  auto kernel = vec16 ? inter ? rotary_kernel<T, 8, true> : rotary_kernel<T, 8, false>
                      : inter ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>;
  kernel<<<(unsigned)n, threads, 0, st>>>(p);
  return launch_status();
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_rotary_append(const pkv_pool* pool, int32_t layer, const void* qkv, int64_t qkv_stride,
                                 int64_t n_tokens, int32_t num_q_heads, const int64_t* positions,
                                 const double* inv_freq, int32_t rotary_dim, int32_t interleaved,
                                 float attention_factor, void* q_out, int64_t q_out_stride_t, int64_t q_out_stride_h,
                                 void* k_out, int64_t k_out_stride_t, int64_t k_out_stride_h, void* v_out,
                                 int64_t v_out_stride_t, int64_t v_out_stride_h, const int64_t* slot_mapping,
                                 int32_t* status_dev, pkv_stream_t stream) {
  if (!pool || n_tokens < 0 || n_tokens > 0x7fffffff || num_q_heads <= 0) return PKV_ERR_INVALID_ARGUMENT;
  const int d = pool->head_dim, hkv = pool->num_kv_heads;
  if (d <= 0 || hkv <= 0 || num_q_heads % hkv || rotary_dim <= 0 || rotary_dim > d || rotary_dim % 2 ||
      (interleaved != 0 && interleaved != 1))
    return PKV_ERR_INVALID_ARGUMENT;
  if (slot_mapping && (layer < 0 || layer >= pool->num_layers || !pool->k || !pool->v || pool->block_size <= 0 ||
                       pool->num_blocks_total <= 0))
    return PKV_ERR_INVALID_ARGUMENT;
  if ((pool->dtype != PKV_F16 && pool->dtype != PKV_BF16) || rotary_dim / 2 > kMaxHalf) return PKV_ERR_UNSUPPORTED;
  const int64_t row = ((int64_t)num_q_heads + 2 * (int64_t)hkv) * d;
  if (qkv_stride < row) return PKV_ERR_INVALID_ARGUMENT;
  if (row > ((int64_t)1 << 31) / d) return PKV_ERR_UNSUPPORTED;  // units are divided in 32 bits
  if (n_tokens == 0) return PKV_OK;
  if (!qkv || !positions || !inv_freq || !q_out) return PKV_ERR_INVALID_ARGUMENT;
  if (!slot_mapping && !k_out) return PKV_ERR_INVALID_ARGUMENT;  // the rotated keys must go somewhere
  RotaryParams p;
  p.qkv = qkv;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.q_out = q_out;
  p.k_out = k_out;
  p.v_out = v_out;
  p.k_pool = pool->k;
  p.v_pool = pool->v;
  p.slots = slot_mapping;
  p.status = status_dev;
  p.qkv_stride = qkv_stride;
  p.q_st = q_out_stride_t, p.q_sh = q_out_stride_h;
  p.k_st = k_out ? k_out_stride_t : 0, p.k_sh = k_out ? k_out_stride_h : 0;
  p.v_st = v_out ? v_out_stride_t : 0, p.v_sh = v_out ? v_out_stride_h : 0;
  p.layer_base = slot_mapping ? (int64_t)layer * pool->num_blocks_total : 0;
  p.factor = attention_factor;
  p.hq = num_q_heads;
  p.hkv = hkv;
  p.d = d;
  p.half = rotary_dim / 2;
  p.bs = pool->block_size;
  p.nbt = pool->num_blocks_total;
  const uintptr_t addr = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
                         reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out) |
                         (slot_mapping ? reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v)
                                       : 0);
  if ((addr & 1) || (reinterpret_cast<uintptr_t>(inv_freq) & 7)) return PKV_ERR_INVALID_ARGUMENT;
  // 16-byte accesses where every row, head and part of a head starts on 16 bytes; else one
  // element at a time.
  const int64_t parts = qkv_stride | p.q_st | p.q_sh | p.k_st | p.k_sh | p.v_st | p.v_sh | d | p.half;
  const bool vec16 = (addr & 15) == 0 && (parts & 7) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return pool->dtype == PKV_F16 ? launch<__half>(p, n_tokens, vec16, interleaved != 0, st)
                                : launch<__nv_bfloat16>(p, n_tokens, vec16, interleaved != 0, st);
}
