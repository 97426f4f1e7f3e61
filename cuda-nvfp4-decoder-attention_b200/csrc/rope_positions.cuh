// Rotary positions of q and k in one launch: a position per token, any
// frequencies, the first R elements of each head, adjacent-pair or half
// layout.  (The reference's RoPE has adjacent pairs of the whole head at
// positions past_length + t: src/rope.cu:18-72.)
//
// Pair m of R / 2 of a token at position p turns by the angle a = p * f_m:
//   y_e = x_e (A cos a) - x_o (A sin a),  y_o = x_e (A sin a) + x_o (A cos a)
// with (e, o) = (2m, 2m + 1) adjacent or (m, m + R/2) half, A the attention
// factor that long-context scalings multiply both with; elements from R on
// are copied.  The angle is formed and reduced in FP64 (the product of an
// integer and an FP32 frequency is exact up to 2^53), so that it is as good at
// position 1e6 as at 1; sine and cosine are FP32, and each output is rounded
// to BF16 once.  At position 0 elements are only scaled by A.
//
// A block takes the tokens of one (token, all heads) group: the (cos, sin)
// pairs of a token are computed once, in shared memory, and used by every
// head.  Bound by HBM: each element is read once and written once.
#pragma once

#include "common.cuh"

namespace nvfp4da {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 1024;  // (cos, sin) pairs a block keeps

struct RopeQkParams {
  const uint16_t* q;  // [B, T, Hq, D] by element strides, last dimension contiguous
  const uint16_t* k;
  uint16_t* q_out;  // contiguous
  uint16_t* k_out;
  int64_t q_stride[3], k_stride[3];  // batch, token, head
  const int64_t* positions;          // [B, T], batch stride pos_stride
  int64_t pos_stride;
  const float* inv_freq;  // [R / 2]
  float factor;
  int64_t rows;  // B * T
  int tokens, q_heads, kv_heads, head_dim, rotary_dim;
  int tokens_per_block;
};

template <int V>
__device__ __forceinline__ void rope_load(const uint16_t* src, uint16_t (&x)[V]) {
  if constexpr (V == 8) *reinterpret_cast<uint4*>(x) = __ldg(reinterpret_cast<const uint4*>(src));
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(x) = __ldg(reinterpret_cast<const uint2*>(src));
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(x) = __ldg(reinterpret_cast<const uint32_t*>(src));
  else x[0] = *src;
}

template <int V>
__device__ __forceinline__ void rope_store(uint16_t* dst, const uint16_t (&x)[V]) {
  if constexpr (V == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(x);
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(x);
  else *dst = x[0];
}

// The pair (xe, xo) turned by (c, s).  s == 0 only scales (an infinity in the
// other element must not reach this one).
__device__ __forceinline__ void rope_turn(float xe, float xo, float2 cs, uint16_t& ye, uint16_t& yo) {
  if (cs.y == 0.0f) {
    ye = f32_to_bf16_bits(__fmul_rn(xe, cs.x));
    yo = f32_to_bf16_bits(__fmul_rn(xo, cs.x));
  } else {
    ye = f32_to_bf16_bits(fmaf(xe, cs.x, -__fmul_rn(xo, cs.y)));
    yo = f32_to_bf16_bits(fmaf(xe, cs.y, __fmul_rn(xo, cs.x)));
  }
}

template <int V, bool ADJACENT>
__global__ void __launch_bounds__(kRopeThreads) rope_qk_kernel(const RopeQkParams p) {
  __shared__ float2 table[kRopeMaxPairs];
  const int pairs = p.rotary_dim / 2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int n_rows = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.rows - row0));
  // Items of V elements (half layout, and adjacent pairs that no 4-byte access
  // covers: V pairs); those past the rotated part are copies.
  constexpr bool kTwo = !ADJACENT || V == 1;  // an item is two pieces
  const int rot = kTwo ? pairs / V : p.rotary_dim / V;
  const int items = rot + (p.head_dim - p.rotary_dim) / V;
  const int heads = p.q_heads + p.kv_heads, total = n_rows * heads * items;
  struct Item {
    alignas(16) uint16_t x[V], z[V];
    uint16_t* dst;  // of x
    int apart;      // elements from x to z; 0: one piece
    int at;         // its first pair in the table; -1: a copy
  };
  auto load = [&](int i, Item& it) {
    const int c = i % items, rh = i / items, hh = rh % heads, r = rh / heads;
    const int64_t row = row0 + r, b = row / p.tokens, t = row % p.tokens;
    const bool is_q = hh < p.q_heads;
    const int h = is_q ? hh : hh - p.q_heads;
    const uint16_t* src = is_q ? p.q + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2]
                               : p.k + b * p.k_stride[0] + t * p.k_stride[1] + h * p.k_stride[2];
    it.dst = is_q ? p.q_out + (row * p.q_heads + h) * p.head_dim : p.k_out + (row * p.kv_heads + h) * p.head_dim;
    int d = 0;
    it.apart = 0;
    it.at = -1;
    if (c >= rot) {
      d = p.rotary_dim + (c - rot) * V;
    } else if constexpr (ADJACENT) {
      d = V == 1 ? 2 * c : c * V;
      it.at = r * pairs + d / 2;
      it.apart = V == 1 ? 1 : 0;
    } else {
      d = c * V;
      it.at = r * pairs + d;
      it.apart = pairs;
    }
    it.dst += d;
    rope_load<V>(src + d, it.x);
    if (kTwo && it.apart) rope_load<V>(src + d + it.apart, it.z);
  };
  auto finish = [&](Item& it) {
    if (it.at >= 0) {
      if constexpr (kTwo) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          rope_turn(bf16_bits_to_f32(it.x[e]), bf16_bits_to_f32(it.z[e]), table[it.at + e], it.x[e], it.z[e]);
        rope_store<V>(it.dst + it.apart, it.z);
      } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e)
          rope_turn(bf16_bits_to_f32(it.x[2 * e]), bf16_bits_to_f32(it.x[2 * e + 1]), table[it.at + e], it.x[2 * e],
                    it.x[2 * e + 1]);
      }
    }
    rope_store<V>(it.dst, it.x);
  };
  // The first item of every thread is on its way while the table is made.
  Item first;
  if (threadIdx.x < total) load(threadIdx.x, first);
  for (int i = threadIdx.x; i < n_rows * pairs; i += kRopeThreads) {
    const int64_t row = row0 + i / pairs;
    const int64_t pos = p.positions[(row / p.tokens) * p.pos_stride + row % p.tokens];
    // a / pi, reduced to [-1, 1]
    const double turns = static_cast<double>(pos) * static_cast<double>(p.inv_freq[i % pairs]) * 0.31830988618379067154;
    float s, c;
    sincospif(static_cast<float>(turns - 2.0 * rint(0.5 * turns)), &s, &c);
    table[i] = make_float2(__fmul_rn(c, p.factor), __fmul_rn(s, p.factor));
  }
  __syncthreads();
  if (threadIdx.x < total) finish(first);
  for (int i = threadIdx.x + kRopeThreads; i < total; i += kRopeThreads) {
    Item it;
    load(i, it);
    finish(it);
  }
}

}  // namespace nvfp4da
