// The quantised KV cache: rows quantised as they are appended, and a window of
// rows read back as BF16.  (No counterpart in the reference, whose cache is
// BF16: src/kv_cache.cu:18-57.)
//
// One row is the D elements of one (sequence, KV head, position).  Formats:
//   E4M3   codes uint8 [B, Hkv, C, D], row scale gamma float32 [B, Hkv, C]:
//            enc = min(448 * (1 / amax), FLT_MAX), 1 for amax = max |x| = 0;
//            gamma = amax * FP32(1/448); code = E4M3_RNE(x * enc);
//            value = code * gamma.
//   NVFP4  every row is one [1, D] matrix of the weight format: packed E2M1
//          uint8 [B, Hkv, C, D/2], UE4M3 block-16 scales uint8 [B, Hkv, C,
//          D/16], gamma float32 [B, Hkv, C]:
//            enc = min(2688 * (1 / amax), FLT_MAX); gamma = amax * FP32(1/2688);
//            beta = UE4M3_RNE(block amax * (enc * FP32(1/6)));
//            code = E2M1_RNE(x * min(1 / (beta * (1 / enc)), FLT_MAX)),
//            0 where beta = 0; value = (code * beta) * gamma.
// Every operation above is one IEEE-rounded FP32 operation; a row is rounded
// to 8 or 4 bits once, when it is written.  (The weight quantiser in
// elementwise.cuh divides 2688 by amax in one rounding; here the reciprocal is
// rounded first, so a value on a rounding boundary may fall to the other side.)
// A row that holds an infinity or NaN is stored with gamma = NaN and zero
// codes: it reads back as NaN throughout, and no code ever is NaN itself.
//
// 8 elements (16 BF16 bytes) per lane, D / 8 lanes of a power-of-two group per
// row, K and V in the same thread: the row maximum is a shuffle reduction and
// nothing is staged.  Both kernels are bound by HBM.
#pragma once

#include <float.h>

#include "common.cuh"

namespace nvfp4da {

constexpr int kKvFmtBf16 = 0, kKvFmtE4m3 = 1, kKvFmtNvfp4 = 2;
constexpr int kKvThreads = 128;

// One of K or V of a quantised cache.
struct KvStore {
  uint8_t* codes;
  uint8_t* block_scales;  // NVFP4 only
  float* row_scales;
};

struct KvAppendParams {
  KvStore k, v;
  const uint16_t* new_k;  // [B, T, Hkv, D] by element strides, last dimension contiguous
  const uint16_t* new_v;
  int64_t k_stride[3], v_stride[3];  // batch, token, head
  int batch, tokens, kv_heads, head_dim;
  int64_t capacity;
  int64_t past_length;          // used when past_lengths == nullptr
  const int64_t* past_lengths;  // device [B]
  const int64_t* counts;        // device [B] or nullptr: tokens t >= counts[b] are not written
  int lanes;                    // lanes per row (power of two >= D / 8)
  int vec_k, vec_v;             // 16-byte loads are aligned
};

struct KvReadParams {
  KvStore k, v;
  uint16_t* out_k;  // [B, Hkv, L, D]
  uint16_t* out_v;
  int batch, kv_heads, head_dim;
  int64_t capacity;
  int64_t length;
  int64_t start;          // used when starts == nullptr
  const int64_t* starts;  // device [B]
  int lanes;
};

// Two FP32 values -> two E4M3 bytes (lo in the low byte), nearest even, saturating.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two FP32 values -> two E2M1 nibbles (lo in the low nibble), nearest even, saturating.
__device__ __forceinline__ uint32_t f32x2_to_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n .reg .b8 b;\n cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n cvt.u32.u8 %0, b;\n}" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two E4M3 bytes (the low 16 bits) -> exact f16x2, low byte in the low half.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two_bytes) {
  uint32_t out;
  asm("{\n .reg .b16 s;\n cvt.u16.u32 s, %1;\n cvt.rn.f16x2.e4m3x2 %0, s;\n}" : "=r"(out) : "r"(two_bytes));
  return out;
}

__device__ __forceinline__ float2 f16x2_to_f32x2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The lane's 8 elements (d0 = 8 * lane in the row) of a row, BF16 pairs.
__device__ __forceinline__ uint4 kv_load8(const uint16_t* row, int d0, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(row + d0));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = static_cast<uint32_t>(row[d0 + 2 * i]) | (static_cast<uint32_t>(row[d0 + 2 * i + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Quantise one row held 8 elements per lane by a group of `lanes` lanes and
// write it.  Every lane of the warp takes part in the shuffles; `live` lanes
// store (d0 < D and the slot exists).
template <int FMT>
__device__ __forceinline__ void kv_quantize_row(const uint4& raw, int lanes, int sub, bool live, const KvStore& st,
                                                int64_t row, int head_dim) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  // max |x| on the bit patterns: for finite values the integer order is the
  // float order, and any infinity or NaN is >= 0x7f80.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  uint32_t pair_top = max(top, __shfl_xor_sync(kFull, top, 1));  // the 16-element block
  top = pair_top;
  for (int o = 2; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
  const bool finite = top < 0x7f80u;
  const float amax = __uint_as_float(top << 16);
  const float range = FMT == kKvFmtE4m3 ? 448.0f : 2688.0f;
  const float enc = amax == 0.0f ? 1.0f : fminf(__fmul_rn(__frcp_rn(amax), range), FLT_MAX);
  const float gamma =
      finite ? __fmul_rn(amax, static_cast<float>(FMT == kKvFmtE4m3 ? 1.0 / 448.0 : 1.0 / 2688.0))
             : __uint_as_float(0x7fc00000u);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  if (FMT == kKvFmtE4m3) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = f32x2_to_e4m3x2(__fmul_rn(x[2 * i], enc), __fmul_rn(x[2 * i + 1], enc));
    if (live)
      *reinterpret_cast<uint2*>(st.codes + row * head_dim + sub * 8) =
          finite ? make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16)) : make_uint2(0u, 0u);
  } else {
    const float bmax = __uint_as_float(pair_top << 16);
    const float mult = __fmul_rn(enc, static_cast<float>(1.0 / 6.0));
    const uint32_t sc = finite ? f32x2_to_e4m3x2(__fmul_rn(bmax, mult), 0.0f) & 0xffu : 0u;
    const float beta = decode_ue4m3(sc);
    uint32_t codes = 0;
    if (beta > 0.0f) {
      const float factor = fminf(__fdiv_rn(1.0f, __fmul_rn(beta, __fdiv_rn(1.0f, enc))), FLT_MAX);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        codes |= f32x2_to_e2m1x2(__fmul_rn(x[2 * i], factor), __fmul_rn(x[2 * i + 1], factor)) << (8 * i);
    }
    if (live) {
      *reinterpret_cast<uint32_t*>(st.codes + row * (head_dim / 2) + sub * 4) = codes;
      if ((sub & 1) == 0) st.block_scales[row * (head_dim / 16) + (sub >> 1)] = static_cast<uint8_t>(sc);
    }
  }
  if (live && sub == 0) st.row_scales[row] = gamma;
}

template <int FMT>
__global__ void __launch_bounds__(kKvThreads) kv_quant_append_kernel(const KvAppendParams p) {
  const int lane = threadIdx.x & 31;
  const int sub = lane & (p.lanes - 1);
  const uint32_t group = (blockIdx.x * kKvThreads + threadIdx.x) / p.lanes;
  const uint32_t total = static_cast<uint32_t>(p.batch) * p.kv_heads * p.tokens;
  // Row order (b, h, t): consecutive groups write consecutive cache rows.
  const uint32_t i = group < total ? group : 0;
  const uint32_t t = i % p.tokens, bh = i / p.tokens, h = bh % p.kv_heads, b = bh / p.kv_heads;
  const int64_t past = p.past_lengths ? p.past_lengths[b] : p.past_length;
  const int64_t slot = past + t;
  bool live = group < total && sub * 8 < p.head_dim && past >= 0 && past < p.capacity && slot < p.capacity;
  if (live && p.counts) live = t < p.counts[b];
  uint4 rk = make_uint4(0, 0, 0, 0), rv = rk;
  if (live) {
    rk = kv_load8(p.new_k + b * p.k_stride[0] + t * p.k_stride[1] + h * p.k_stride[2], sub * 8, p.vec_k);
    rv = kv_load8(p.new_v + b * p.v_stride[0] + t * p.v_stride[1] + h * p.v_stride[2], sub * 8, p.vec_v);
  }
  const int64_t row = static_cast<int64_t>(bh) * p.capacity + slot;
  kv_quantize_row<FMT>(rk, p.lanes, sub, live, p.k, row, p.head_dim);
  kv_quantize_row<FMT>(rv, p.lanes, sub, live, p.v, row, p.head_dim);
}

// 8 elements of a stored row, FP32: (code * beta) * gamma, or code * gamma.
template <int FMT>
__device__ __forceinline__ void kv_decode8(const KvStore& st, int64_t row, int d0, int head_dim, float (&x)[8]) {
  const float gamma = __ldg(st.row_scales + row);
  if (FMT == kKvFmtE4m3) {
    const uint2 c = __ldg(reinterpret_cast<const uint2*>(st.codes + row * head_dim + d0));
    const uint32_t h[4] = {e4m3x2_to_f16x2(c.x & 0xffffu), e4m3x2_to_f16x2(c.x >> 16), e4m3x2_to_f16x2(c.y & 0xffffu),
                           e4m3x2_to_f16x2(c.y >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = f16x2_to_f32x2(h[i]);
      x[2 * i] = __fmul_rn(f.x, gamma);
      x[2 * i + 1] = __fmul_rn(f.y, gamma);
    }
  } else {
    const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(st.codes + row * (head_dim / 2) + d0 / 2));
    const float beta = decode_ue4m3(__ldg(st.block_scales + row * (head_dim / 16) + d0 / 16));
    uint32_t h[4];
    e2m1x8_to_f16x2x4(c, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = f16x2_to_f32x2(h[i]);
      x[2 * i] = __fmul_rn(__fmul_rn(f.x, beta), gamma);
      x[2 * i + 1] = __fmul_rn(__fmul_rn(f.y, beta), gamma);
    }
  }
}

__device__ __forceinline__ uint4 kv_pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = static_cast<uint32_t>(f32_to_bf16_bits(x[2 * i])) |
           (static_cast<uint32_t>(f32_to_bf16_bits(x[2 * i + 1])) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int FMT>
__global__ void __launch_bounds__(kKvThreads) kv_quant_read_kernel(const KvReadParams p) {
  const int sub = threadIdx.x & (p.lanes - 1);
  const uint32_t group = (blockIdx.x * kKvThreads + threadIdx.x) / p.lanes;
  const uint32_t len = static_cast<uint32_t>(p.length);
  const uint32_t total = static_cast<uint32_t>(p.batch) * p.kv_heads * len;
  if (group >= total || sub * 8 >= p.head_dim) return;
  const uint32_t j = group % len, bh = group / len, b = bh / p.kv_heads;
  const int64_t start = p.starts ? p.starts[b] : p.start;
  // Rows outside the cache read as zeros.
  const bool inside = start > -static_cast<int64_t>(len) && start < p.capacity && start + j >= 0 && start + j < p.capacity;
  float k[8] = {}, v[8] = {};
  if (inside) {
    const int64_t row = static_cast<int64_t>(bh) * p.capacity + start + j;
    kv_decode8<FMT>(p.k, row, sub * 8, p.head_dim, k);
    kv_decode8<FMT>(p.v, row, sub * 8, p.head_dim, v);
  }
  const int64_t dst = static_cast<int64_t>(group) * p.head_dim + sub * 8;
  *reinterpret_cast<uint4*>(p.out_k + dst) = kv_pack8(k);
  *reinterpret_cast<uint4*>(p.out_v + dst) = kv_pack8(v);
}

}  // namespace nvfp4da
