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
// Append: a lane takes one 16-element block of a row's K and of its V, D / 16
// lanes (a power of two) a row: the row maximum is a shuffle reduction over
// few lanes, and the divisions of the scales are shared by 16 elements (with 8
// per lane they were half of the instructions, which bound the kernel).  Read:
// 8 elements per lane, so that 16-byte stores of a warp are contiguous, and
// several rows of K and V in flight per thread.  Measured: 32,768 positions x
// 24 heads of E4M3 read back, with an append of 8, in 99 to 104 us (5.9 to 6.2
// TB/s, 0.90 to 0.94 of a copy).  Where the cache stays in L2 the instructions
// bound both: 8,192 tokens x 6 heads to NVFP4 rows in 12 us (issue slots 67 %
// busy, DRAM 26 %), and back in 10 us (62 %).
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
  int lanes;                    // lanes per row (power of two >= D / 16)
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
  int lanes;              // lanes per row (power of two >= D / 8)
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

// A lane's 16 elements of a row, BF16 pairs.
__device__ __forceinline__ void kv_load16(const uint16_t* src, bool vec, uint32_t (&w)[8]) {
  if (vec) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(src)), b = __ldg(reinterpret_cast<const uint4*>(src) + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i] = static_cast<uint32_t>(src[2 * i]) | (static_cast<uint32_t>(src[2 * i + 1]) << 16);
  }
}

// Quantise one row held 16 elements per lane by a group of `lanes` lanes and
// write it.  Every lane of the warp takes part in the shuffles; `live` lanes
// store (16 sub < D and the slot exists).
template <int FMT>
__device__ __forceinline__ void kv_quantize_row(const uint32_t (&w)[8], int lanes, int sub, bool live,
                                                const KvStore& st, int64_t row, int head_dim) {
  // max |x| on the bit patterns: for finite values the integer order is the
  // float order, and any infinity or NaN is >= 0x7f80.
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = max(lo, w[i] & 0x7fffu);
    hi = max(hi, w[i] & 0x7fff0000u);
  }
  const uint32_t block_top = max(lo, hi >> 16);
  uint32_t top = block_top;
  for (int o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
  const bool finite = top < 0x7f80u;
  const float amax = __uint_as_float(top << 16);
  const float range = FMT == kKvFmtE4m3 ? 448.0f : 2688.0f;
  const float enc = amax == 0.0f ? 1.0f : fminf(__fmul_rn(__frcp_rn(amax), range), FLT_MAX);
  const float gamma =
      finite ? __fmul_rn(amax, static_cast<float>(FMT == kKvFmtE4m3 ? 1.0 / 448.0 : 1.0 / 2688.0))
             : __uint_as_float(0x7fc00000u);
  auto lower = [&](int i) { return __uint_as_float(w[i] << 16); };
  auto upper = [&](int i) { return __uint_as_float(w[i] & 0xffff0000u); };
  if (FMT == kKvFmtE4m3) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = f32x2_to_e4m3x2(__fmul_rn(lower(2 * i), enc), __fmul_rn(upper(2 * i), enc));
      const uint32_t b = f32x2_to_e4m3x2(__fmul_rn(lower(2 * i + 1), enc), __fmul_rn(upper(2 * i + 1), enc));
      c[i] = finite ? a | (b << 16) : 0u;
    }
    if (live) *reinterpret_cast<uint4*>(st.codes + row * head_dim + sub * 16) = make_uint4(c[0], c[1], c[2], c[3]);
  } else {
    const float bmax = __uint_as_float(block_top << 16);
    const float mult = __fmul_rn(enc, static_cast<float>(1.0 / 6.0));
    const uint32_t sc = finite ? f32x2_to_e4m3x2(__fmul_rn(bmax, mult), 0.0f) & 0xffu : 0u;
    const float beta = decode_ue4m3(sc);
    uint32_t c[2] = {0u, 0u};
    if (beta > 0.0f) {
      const float factor = fminf(__frcp_rn(__fmul_rn(beta, __frcp_rn(enc))), FLT_MAX);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        c[i / 4] |= f32x2_to_e2m1x2(__fmul_rn(lower(i), factor), __fmul_rn(upper(i), factor)) << (8 * (i % 4));
    }
    if (live) {
      *reinterpret_cast<uint2*>(st.codes + row * (head_dim / 2) + sub * 8) = make_uint2(c[0], c[1]);
      st.block_scales[row * (head_dim / 16) + sub] = static_cast<uint8_t>(sc);
    }
  }
  if (live && sub == 0) st.row_scales[row] = gamma;
}

// Grid (rows of T, B * Hkv).
template <int FMT>
__global__ void __launch_bounds__(kKvThreads) kv_quant_append_kernel(const KvAppendParams p) {
  const int sub = threadIdx.x & (p.lanes - 1);
  const int t = blockIdx.x * (kKvThreads / p.lanes) + threadIdx.x / p.lanes;
  const int h = blockIdx.y % p.kv_heads, b = blockIdx.y / p.kv_heads;
  const int64_t past = p.past_lengths ? p.past_lengths[b] : p.past_length;
  const int64_t slot = past + t;
  bool live = t < p.tokens && sub * 16 < p.head_dim && past >= 0 && past < p.capacity && slot < p.capacity;
  if (live && p.counts) live = t < p.counts[b];
  uint32_t wk[8] = {}, wv[8] = {};
  if (live) {
    kv_load16(p.new_k + b * p.k_stride[0] + t * p.k_stride[1] + h * p.k_stride[2] + sub * 16, p.vec_k, wk);
    kv_load16(p.new_v + b * p.v_stride[0] + t * p.v_stride[1] + h * p.v_stride[2] + sub * 16, p.vec_v, wv);
  }
  const int64_t row = static_cast<int64_t>(blockIdx.y) * p.capacity + slot;
  kv_quantize_row<FMT>(wk, p.lanes, sub, live, p.k, row, p.head_dim);
  kv_quantize_row<FMT>(wv, p.lanes, sub, live, p.v, row, p.head_dim);
}

// 8 elements of a stored row as they are in memory (zeros: a row of zeros).
template <int FMT>
struct KvRaw {
  uint32_t c[FMT == kKvFmtE4m3 ? 2 : 1] = {};
  uint32_t beta = 0;
  float gamma = 0.0f;
};

template <int FMT>
__device__ __forceinline__ KvRaw<FMT> kv_fetch8(const KvStore& st, int64_t row, int d0, int head_dim) {
  KvRaw<FMT> r;
  r.gamma = __ldg(st.row_scales + row);
  if constexpr (FMT == kKvFmtE4m3) {
    const uint2 c = __ldg(reinterpret_cast<const uint2*>(st.codes + row * head_dim + d0));
    r.c[0] = c.x;
    r.c[1] = c.y;
  } else {
    r.c[0] = __ldg(reinterpret_cast<const uint32_t*>(st.codes + row * (head_dim / 2) + d0 / 2));
    r.beta = __ldg(st.block_scales + row * (head_dim / 16) + d0 / 16);
  }
  return r;
}

// Their FP32 values: (code * beta) * gamma, or code * gamma.
template <int FMT>
__device__ __forceinline__ void kv_decode8(const KvRaw<FMT>& r, float (&x)[8]) {
  uint32_t h[4];
  if constexpr (FMT == kKvFmtE4m3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = e4m3x2_to_f16x2(r.c[i / 2] >> (16 * (i % 2)) & 0xffffu);
  } else {
    e2m1x8_to_f16x2x4(r.c[0], h);
  }
  const float beta = FMT == kKvFmtNvfp4 ? decode_ue4m3(r.beta) : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = f16x2_to_f32x2(h[i]);
    x[2 * i] = __fmul_rn(FMT == kKvFmtNvfp4 ? __fmul_rn(f.x, beta) : f.x, r.gamma);
    x[2 * i + 1] = __fmul_rn(FMT == kKvFmtNvfp4 ? __fmul_rn(f.y, beta) : f.y, r.gamma);
  }
}

template <int FMT>
__device__ __forceinline__ void kv_decode8(const KvStore& st, int64_t row, int d0, int head_dim, float (&x)[8]) {
  kv_decode8<FMT>(kv_fetch8<FMT>(st, row, d0, head_dim), x);
}

__device__ __forceinline__ uint4 kv_pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Grid (rows of the window, B * Hkv); a thread takes kKvReadRows rows.
constexpr int kKvReadRows = 4;

template <int FMT>
__global__ void __launch_bounds__(kKvThreads) kv_quant_read_kernel(const KvReadParams p) {
  const int sub = threadIdx.x & (p.lanes - 1), d0 = sub * 8;
  if (d0 >= p.head_dim) return;
  const int step = kKvThreads / p.lanes;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * step * kKvReadRows + threadIdx.x / p.lanes;
  const int64_t start = p.starts ? p.starts[blockIdx.y / p.kv_heads] : p.start;
  // Rows outside the cache read as zeros.
  const int64_t first = start > -p.length && start < p.capacity ? start : p.capacity;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * p.capacity + first;
  KvRaw<FMT> k[kKvReadRows], v[kKvReadRows];
#pragma unroll
  for (int i = 0; i < kKvReadRows; ++i) {
    const int64_t j = j0 + i * step;
    if (j < p.length && first + j >= 0 && first + j < p.capacity) {
      k[i] = kv_fetch8<FMT>(p.k, row0 + j, d0, p.head_dim);
      v[i] = kv_fetch8<FMT>(p.v, row0 + j, d0, p.head_dim);
    }
  }
#pragma unroll
  for (int i = 0; i < kKvReadRows; ++i) {
    const int64_t j = j0 + i * step;
    if (j >= p.length) return;
    const int64_t dst = (static_cast<int64_t>(blockIdx.y) * p.length + j) * p.head_dim + d0;
    float x[8];
    kv_decode8<FMT>(k[i], x);
    *reinterpret_cast<uint4*>(p.out_k + dst) = kv_pack8(x);
    kv_decode8<FMT>(v[i], x);
    *reinterpret_cast<uint4*>(p.out_v + dst) = kv_pack8(x);
  }
}

}  // namespace nvfp4da
