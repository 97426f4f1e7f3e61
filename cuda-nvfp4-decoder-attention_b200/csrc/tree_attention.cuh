// Attention of a tree of drafted tokens over a BF16, E4M3 or NVFP4 cache: the
// general kernel and the combine of split partials.
//
// The cache [B, Hkv, C, D] holds P_b committed positions of sequence b and,
// from slot P_b on, its T drafted tokens in any order in which ancestors come
// first.  Query head h of drafted token t reads KV head h / (Hq / Hkv) and
// sees key j iff j < P_b, or j = P_b + u with u < T and mask[b, t, u] (without
// a mask: u <= t, the causal chain):
//   s_j = (q . k_j) / sqrt(D),  ctx = sum_j e^{s_j} v_j / sum_j e^{s_j},
// zeros for a query that sees nothing.  Slots at or past P_b + T and keys that
// a query does not see never reach its result, whatever they hold.  With
// T = 1 this is single-token decode.  (The reference attends causally over
// BF16: src/gqa_attention_cached.cu:93-337.)
//
// Sums, maxima and the softmax are FP32; quantised rows are used as the values
// they stand for, without a rounding to BF16.
#pragma once

#include <math.h>

#include "common.cuh"
#include "kv_quant.cuh"

namespace nvfp4da {

struct TreeAttnParams {
  const uint16_t* q;  // [B, T, Hq, D]
  KvStore k, v;       // codes: BF16 rows (as bytes) for a BF16 cache
  const uint8_t* mask;  // [B, T, T] truth values by mask_stride over b (0: one for all), or nullptr
  int64_t mask_stride;
  uint16_t* ctx;   // [B, T, Hq, D]
  float* partials; // [B*T*Hq][splits][D + 2]: o (unnormalised), m, l
  int batch, tokens, q_heads, kv_heads, head_dim;
  int64_t capacity;
  int64_t past_length;  // used when past_lengths == nullptr
  const int64_t* past_lengths;
  float scale;  // 1 / sqrt(D)
  int splits;
  int64_t split_len;
  int lanes;  // lanes per key (power of two >= D / 8)
};

// P_b clamped so that the drafted slots lie in the cache.
__device__ __forceinline__ int64_t tree_past(const int64_t* past_lengths, int64_t past_length, int b, int64_t capacity) {
  const int64_t p = past_lengths ? past_lengths[b] : past_length;
  return p < 0 ? 0 : (p > capacity ? capacity : p);
}

__device__ __forceinline__ bool tree_sees(const uint8_t* mask_row, int t, int64_t u) {
  return u < 0 || (mask_row ? mask_row[u] != 0 : u <= t);
}

template <int FMT>
__device__ __forceinline__ void tree_load8(const KvStore& st, int64_t row, int d0, int head_dim, float (&x)[8]) {
  if (FMT == kKvFmtBf16) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(st.codes + (row * head_dim + d0) * 2));
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(a[i] << 16);
      x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  } else {
    kv_decode8<FMT>(st, row, d0, head_dim, x);
  }
}

constexpr int kTreeWarps = 4;

// Grid (splits, ceil(group * T / 4), B * Hkv): one warp per query row and
// split, `lanes` lanes per key, 32 / lanes keys at a time, every lane 8
// elements of the head.  Every row reads the keys again (from L2): this kernel
// serves the head dimensions the streaming kernel does not.
template <int FMT>
__global__ void __launch_bounds__(kTreeWarps * 32) tree_attn_general_kernel(const TreeAttnParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = p.q_heads / p.kv_heads;
  const int n = blockIdx.y * kTreeWarps + warp;
  if (n >= group * p.tokens) return;
  const int b = blockIdx.z / p.kv_heads, kvh = blockIdx.z % p.kv_heads;
  const int t = n / group, h = kvh * group + n % group;
  const int sub = lane & (p.lanes - 1), d0 = sub * 8;
  const bool has = d0 < p.head_dim;
  const int64_t past = tree_past(p.past_lengths, p.past_length, b, p.capacity);
  const int64_t end = min(past + p.tokens, p.capacity);
  const int64_t j0 = blockIdx.x * p.split_len, j1 = min(j0 + p.split_len, end);
  const uint8_t* mask_row = p.mask ? p.mask + b * p.mask_stride + static_cast<int64_t>(t) * p.tokens : nullptr;
  const int64_t out_row = (static_cast<int64_t>(b) * p.tokens + t) * p.q_heads + h;
  const int64_t row0 = static_cast<int64_t>(blockIdx.z) * p.capacity;

  float q[8] = {}, acc[8] = {};
  if (has) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p.q + out_row * p.head_dim + d0));
    const uint32_t a[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[2 * i] = __uint_as_float(a[i] << 16) * p.scale;
      q[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u) * p.scale;
    }
  }
  float m = -INFINITY, l = 0.0f;
  const int step = 32 / p.lanes;
  for (int64_t base = j0; base < j1; base += step) {
    const int64_t j = base + lane / p.lanes;
    const bool sees = j < j1 && tree_sees(mask_row, t, j - past);
    float k[8] = {}, v[8] = {};
    if (sees && has) {
      tree_load8<FMT>(p.k, row0 + j, d0, p.head_dim, k);
      tree_load8<FMT>(p.v, row0 + j, d0, p.head_dim, v);
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(q[i], k[i], s);
    for (int o = 1; o < p.lanes; o <<= 1) s += __shfl_xor_sync(kFull, s, o);
    if (!sees || s == -INFINITY) continue;  // uniform in the group of lanes; no shuffle below
    const float m_new = fmaxf(m, s);
    const float alpha = m == -INFINITY ? 0.0f : expf(m - m_new), e = expf(s - m_new);
    l = fmaf(l, alpha, e);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(acc[i], alpha, e * v[i]);
    m = m_new;
  }
  __syncwarp();
  for (int o = p.lanes; o < 32; o <<= 1) {  // merge the groups of lanes
    const float m2 = __shfl_xor_sync(kFull, m, o), mx = fmaxf(m, m2);
    const float f = m == -INFINITY ? 0.0f : expf(m - mx), f2 = m2 == -INFINITY ? 0.0f : expf(m2 - mx);
    l = l * f + __shfl_xor_sync(kFull, l, o) * f2;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = acc[i] * f + __shfl_xor_sync(kFull, acc[i], o) * f2;
    m = mx;
  }
  if (lane >= p.lanes || !has) return;
  if (p.splits == 1) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = l == 0.0f ? 0.0f : __fdiv_rn(acc[i], l);
    *reinterpret_cast<uint4*>(p.ctx + out_row * p.head_dim + d0) = kv_pack8(o);
    return;
  }
  float* dst = p.partials + (out_row * p.splits + blockIdx.x) * (p.head_dim + 2);
#pragma unroll
  for (int i = 0; i < 8; ++i) dst[d0 + i] = acc[i];
  if (d0 == 0) {
    dst[p.head_dim] = m;
    dst[p.head_dim + 1] = l;
  }
}

// One warp per query row: its splits' partials, joined in split order.
__global__ void __launch_bounds__(128) tree_combine_kernel(const TreeAttnParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(p.batch) * p.tokens * p.q_heads) return;
  const float* base = p.partials + row * p.splits * (p.head_dim + 2);
  float mx = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) mx = fmaxf(mx, base[s * (p.head_dim + 2) + p.head_dim]);
  mx = warp_max_f32(mx);
  float l = 0.0f, o[8] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float* src = base + s * (p.head_dim + 2);
    const float ms = src[p.head_dim];
    if (ms == -INFINITY && src[p.head_dim + 1] == 0.0f) continue;
    const float f = expf(ms - mx);
    l = fmaf(src[p.head_dim + 1], f, l);
    for (int i = 0, d = lane; d < p.head_dim; ++i, d += 32) o[i] = fmaf(src[d], f, o[i]);
  }
  for (int i = 0, d = lane; d < p.head_dim; ++i, d += 32)
    p.ctx[row * p.head_dim + d] = f32_to_bf16_bits(l == 0.0f ? 0.0f : __fdiv_rn(o[i], l));
}

}  // namespace nvfp4da
