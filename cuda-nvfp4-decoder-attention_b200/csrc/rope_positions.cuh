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
// A block takes one token (several where heads are few): the sines and cosines
// are computed once per token, in shared memory, laid out so that one 16-byte
// load serves two FP32x2 operations.  Each element is read once and written once,
// with its first loads on their way while the table is made.
// Measured: 8,192 tokens x 30 heads x 128 elements, 126 MB, in 27 us (4.7
// TB/s, 0.72 of a copy); instructions issue in 80 % of the cycles there: 310 a
// thread for its one item of 16 elements, most of them what a block of one token
// sets up (divisions of indices, the table).  A single token: 7.8 us, the
// launch.
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
  uint32_t rows;  // B * T, below 2^31 (32-bit divisions: 64-bit ones took longer than the memory)
  uint32_t tokens;
  int q_heads, kv_heads, head_dim, rotary_dim;
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

__device__ __forceinline__ float2 rope_mul2(float2 a, float2 b) {
  float2 c;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n"
      " mov.b64 {%0, %1}, z;\n}" : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ float2 rope_fma2(float2 a, float2 b, float2 d) {
  float2 c;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 w, {%6, %7};\n"
      " fma.rn.f32x2 z, x, y, w;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(d.x), "f"(d.y));
  return c;
}
__device__ __forceinline__ uint32_t rope_pack(float2 v) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
  return r;
}
__device__ __forceinline__ float2 rope_unpack(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Items of V elements, or where an item is two pieces (half layout; adjacent
// pairs that no 4-byte access covers) V pairs; those past the rotated part are
// copies.
template <int V, bool ADJACENT>
__global__ void __launch_bounds__(kRopeThreads) rope_qk_kernel(const RopeQkParams p) {
  constexpr bool kTwo = !ADJACENT || V == 1;
  constexpr bool kPairs = kTwo && V > 1;  // a table entry serves two pairs: {c0, c1, s0, s1}, else {c, s, -s, c}
  constexpr int W = kTwo ? V : V / 2;     // pairs per item
  __shared__ float4 table[kRopeMaxPairs];
  __shared__ unsigned char at_zero[kRopeMaxPairs];  // tokens at position 0: only scaled
  const int pairs = p.rotary_dim / 2;
  const uint32_t row0 = blockIdx.x * static_cast<uint32_t>(p.tokens_per_block);
  const int n_rows = static_cast<int>(min(static_cast<uint32_t>(p.tokens_per_block), p.rows - row0));
  const int rot = kTwo ? pairs / V : p.rotary_dim / V;
  const int items = rot + (p.head_dim - p.rotary_dim) / V;
  const int heads = p.q_heads + p.kv_heads;
  // Threads as tx items by ty heads.
  const int tx = min(items, kRopeThreads), ty = kRopeThreads / tx;
  const int y0 = threadIdx.x / tx, c0 = threadIdx.x - y0 * tx;
  const uint32_t b0 = row0 / p.tokens, t0 = row0 - b0 * p.tokens;
  struct Item {
    alignas(16) uint16_t x[V];
    alignas(16) uint16_t z[V];
    uint16_t* dst;
    int r;
  };
  auto load = [&](int y, int c, Item& it) {
    int r = 0, hh = y;
    uint32_t row = row0, b = b0, t = t0;
    if (n_rows > 1) {
      r = y / heads;
      hh = y - r * heads;
      row += r;
      b = row / p.tokens;
      t = row - b * p.tokens;
    }
    const bool is_q = hh < p.q_heads;
    const int h = is_q ? hh : hh - p.q_heads;
    const int d = c >= rot ? p.rotary_dim + (c - rot) * V : (ADJACENT && V == 1 ? 2 * c : c * V);
    const uint16_t* src = (is_q ? p.q + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2]
                                : p.k + b * p.k_stride[0] + t * p.k_stride[1] + h * p.k_stride[2]) + d;
    it.dst = (is_q ? p.q_out + (static_cast<int64_t>(row) * p.q_heads + h) * p.head_dim
                   : p.k_out + (static_cast<int64_t>(row) * p.kv_heads + h) * p.head_dim) + d;
    it.r = r;
    rope_load<V>(src, it.x);
    if (kTwo && c < rot) rope_load<V>(src + (ADJACENT ? 1 : pairs), it.z);
  };
  auto finish = [&](int c, Item& it) {
    if (c < rot) {
      const float4* entry = table + it.r * pairs + c;
      const bool turn = !at_zero[it.r];
      if constexpr (kPairs) {
        uint32_t *x = reinterpret_cast<uint32_t*>(it.x), *z = reinterpret_cast<uint32_t*>(it.z);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float4 u = entry[e * rot];
          const float2 a = rope_unpack(x[e]), o = rope_unpack(z[e]), cs = make_float2(u.x, u.y);
          float2 ya = rope_mul2(a, cs), yo = rope_mul2(o, cs);
          if (turn) {
            ya = rope_fma2(o, make_float2(-u.z, -u.w), ya);
            yo = rope_fma2(a, make_float2(u.z, u.w), yo);
          }
          x[e] = rope_pack(ya);
          z[e] = rope_pack(yo);
        }
      } else if constexpr (kTwo) {
        const float4 u = entry[0];
        const float a = bf16_bits_to_f32(it.x[0]), o = bf16_bits_to_f32(it.z[0]);
        it.x[0] = f32_to_bf16_bits(turn ? fmaf(o, u.z, __fmul_rn(a, u.x)) : __fmul_rn(a, u.x));
        it.z[0] = f32_to_bf16_bits(turn ? fmaf(a, u.y, __fmul_rn(o, u.x)) : __fmul_rn(o, u.x));
      } else {
        uint32_t* x = reinterpret_cast<uint32_t*>(it.x);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float4 u = entry[e * rot];
          const float2 v = rope_unpack(x[e]);
          x[e] = rope_pack(turn ? rope_fma2(make_float2(v.y, v.y), make_float2(u.z, u.w),
                                            rope_mul2(make_float2(v.x, v.x), make_float2(u.x, u.y)))
                                : rope_mul2(v, make_float2(u.x, u.x)));
        }
      }
      if constexpr (kTwo) rope_store<V>(it.dst + (ADJACENT ? 1 : pairs), it.z);
    }
    rope_store<V>(it.dst, it.x);
  };
  const int last = n_rows * heads;
  const bool busy = y0 < ty;
  Item first;
  if (busy && y0 < last && c0 < items) load(y0, c0, first);
  for (int i = threadIdx.x; i < n_rows * pairs; i += kRopeThreads) {
    const int r = n_rows == 1 ? 0 : i / pairs, m = i - r * pairs;
    const uint32_t row = row0 + r, b = row / p.tokens;
    const int64_t pos = p.positions[b * p.pos_stride + (row - b * p.tokens)];
    // a / pi, reduced to [-1, 1]
    const double turns = static_cast<double>(pos) * static_cast<double>(p.inv_freq[m]) * 0.31830988618379067154;
    float s, c;
    sincospif(static_cast<float>(turns - 2.0 * rint(0.5 * turns)), &s, &c);
    c = __fmul_rn(c, p.factor);
    s = __fmul_rn(s, p.factor);
    const int e = m % W, item = m / W;
    if constexpr (kPairs) {
      float* u = reinterpret_cast<float*>(table + r * pairs + e / 2 * rot + item) + e % 2;
      u[0] = c;
      u[2] = s;
    } else {
      table[r * pairs + e * rot + item] = make_float4(c, s, -s, c);
    }
    if (m == 0) at_zero[r] = pos == 0;
  }
  __syncthreads();
  if (!busy) return;
  for (int y = y0; y < last; y += ty)
    for (int c = c0; c < items; c += tx) {
      if (y != y0 || c != c0) load(y, c, first);
      finish(c, first);
    }
}

}  // namespace nvfp4da
