// Attention through a block table for the head dimensions (multiples of 16) and
// batches that the streaming kernel does not take.  Semantics: tree_attention.cuh,
// paged_kv.cuh.
//
// Grid (splits, passes of 16 query rows, B * Hkv), four warps a CTA, several CTAs an
// SM: their loads and their arithmetic overlap one another.  A tile of 64 keys of K
// and V comes row by row, through the table, into shared memory: BF16 as it is,
// codes (times the NVFP4 block scale) as FP16, exact.
// Each warp takes 16 keys of it:
//   S[q, key] = Q K^T      mma.m16n8k16, exact products; times K's row scale
//   O[q, d]  += P V        mma.m16n8k8, TF32: P times V's row scale is rounded to 11
//                          bits, in the exponents of FP32, whatever the scales are;
//                          V is exact
// with the k of P V permuted so that the scores' registers are P's operand.  The
// running maximum, sums and o are FP32; the warps' parts are joined in shared memory,
// the splits' by tree_combine_kernel.  Infinities and NaN of V in drafted rows become
// 0 in the tile (0 * NaN would reach queries that do not see the row) and are added
// at the end for the queries that do.
//
// 64 sequences x 6 heads, 1,024 to 8,191 positions, head_dim 96, one token x 4 heads:
// BF16 247 us, E4M3 225, NVFP4 212 (floors 106, 55, 32; a warp per query row with
// scalar products, as over whole caches, took 1.2 ms for a smaller call).  Bound by
// instructions and the latency between them: a quarter of a tile's 16 query rows is
// in use, issue slots 42 %.
#pragma once

#include <math.h>

#include "common.cuh"
#include "kv_quant.cuh"
#include "paged_kv.cuh"
#include "tree_attention.cuh"

namespace nvfp4da {

constexpr int kPgenWarps = 4, kPgenThreads = kPgenWarps * 32, kPgenTile = 64, kPgenRows = 16;

// Shared memory: K and V [64][D + 8] (later the warps' o), Q [16][D + 8], BF16.
template <int KS>
constexpr uint32_t pgen_smem() { return (2 * kPgenTile + kPgenRows) * (16 * KS + 8) * 2; }

__device__ __forceinline__ void pgen_ldsm4(const uint16_t* at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(at)));
}
__device__ __forceinline__ uint32_t pgen_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float pgen_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 elements of a row of K or V as they are in memory; zeros: a row of zeros.
template <int FMT>
struct PgenRaw {
  uint4 c[FMT == kKvFmtBf16 ? 2 : 1];
  uint32_t beta;
};

template <int FMT>
__device__ __forceinline__ PgenRaw<FMT> pgen_fetch16(const KvStore& st, int64_t row, int d0, int head_dim) {
  PgenRaw<FMT> r;
  r.c[0] = make_uint4(0u, 0u, 0u, 0u);
  r.beta = 0u;
  if constexpr (FMT == kKvFmtBf16) r.c[1] = r.c[0];
  if (row < 0) return r;
  if constexpr (FMT == kKvFmtBf16) {
    const uint4* src = reinterpret_cast<const uint4*>(st.codes + (row * head_dim + d0) * 2);
    r.c[0] = __ldg(src);
    r.c[1] = __ldg(src + 1);
  } else if constexpr (FMT == kKvFmtE4m3) {
    r.c[0] = __ldg(reinterpret_cast<const uint4*>(st.codes + row * head_dim + d0));
  } else {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(st.codes + row * (head_dim / 2) + d0 / 2));
    r.c[0].x = a.x;
    r.c[0].y = a.y;
    r.beta = __ldg(st.block_scales + row * (head_dim / 16) + d0 / 16);
  }
  return r;
}

// Their values without the row scale: BF16 pairs, or codes (times the block scale) as FP16 pairs, exact.
template <int FMT>
__device__ __forceinline__ void pgen_decode16(const PgenRaw<FMT>& r, uint32_t (&w)[8]) {
  if constexpr (FMT == kKvFmtBf16) {
    w[0] = r.c[0].x, w[1] = r.c[0].y, w[2] = r.c[0].z, w[3] = r.c[0].w;
    w[4] = r.c[1].x, w[5] = r.c[1].y, w[6] = r.c[1].z, w[7] = r.c[1].w;
  } else if constexpr (FMT == kKvFmtE4m3) {
    const uint32_t c[4] = {r.c[0].x, r.c[0].y, r.c[0].z, r.c[0].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = e4m3x2_to_f16x2(c[i / 2] >> (16 * (i % 2)) & 0xffffu);
  } else {
    const uint32_t beta = e4m3x2_to_f16x2(r.beta * 0x101u);
    uint32_t lo[4], hi[4];
    e2m1x8_to_f16x2x4(r.c[0].x, lo);
    e2m1x8_to_f16x2x4(r.c[0].y, hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(w[i]) : "r"(lo[i]), "r"(beta));
      asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(w[4 + i]) : "r"(hi[i]), "r"(beta));
    }
  }
}

// Both halves of a word of theirs in FP32.
template <int FMT>
__device__ __forceinline__ float2 pgen_pair(uint32_t w) {
  if constexpr (FMT == kKvFmtBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return f16x2_to_f32x2(w);
}

// The halves of w that are infinities or NaN become 0; returns whether there was one.
template <int FMT>
__device__ __forceinline__ bool pgen_finite(uint32_t& w) {
  constexpr uint32_t e = FMT == kKvFmtBf16 ? 0x7f80u : 0x7c00u;
  const bool lo = (w & e) == e, hi = (w >> 16 & e) == e;
  if (lo) w &= 0xffff0000u;
  if (hi) w &= 0x0000ffffu;
  return lo || hi;
}

// Four CTAs an SM up to head_dim 128 (8 x 26,000 positions, head_dim 96: E4M3 206 -> 185 us, NVFP4 192 -> 165); with
// five, or three of larger heads of codes, registers spill.  At 112 and 128 four spill too (bytes stored a thread: BF16
// 360 and 436, E4M3 76 and 72, NVFP4 0 and 28), which costs BF16 and E4M3 at 112 dearly: 64 sequences of 1,024 to 8,191
// positions, head_dim 96 / 112, BF16 247 / 611 us, E4M3 225 / 452, NVFP4 212 / 251.  Three there were not tried.  BF16
// at head_dim 192: three 529 us, two 689.
template <int FMT, int KS>
__global__ void __launch_bounds__(kPgenThreads, KS <= 8 ? 4 : FMT == kKvFmtBf16 ? 3 : 1) paged_attn_general_kernel(const TreeAttnParams p, const PagedView pg) {
  constexpr int D = 16 * KS, kStride = D + 8;  // elements: rows 4 banks apart, modulo 8
  constexpr bool kQuant = FMT != kKvFmtBf16;
  extern __shared__ __align__(16) uint8_t pgen_raw[];
  uint16_t* sk = reinterpret_cast<uint16_t*>(pgen_raw);
  uint16_t* sv = sk + kPgenTile * kStride;
  uint16_t* sq = sv + kPgenTile * kStride;
  float* so = reinterpret_cast<float*>(pgen_raw);  // [warp][16][D], when the tiles are done
  __shared__ int s_row[3][kPgenTile];              // rows of the pool of this tile and the next two, -1: no such key
  __shared__ float s_kr[kPgenTile], s_vr[kPgenTile], s_q[kPgenRows];
  __shared__ float s_m[kPgenWarps][kPgenRows], s_l[kPgenWarps][kPgenRows];
  __shared__ int s_wild;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tq = lane & 3;
  const int group = p.q_heads / p.kv_heads, nq = group * p.tokens;
  const int b = blockIdx.z / p.kv_heads, kvh = blockIdx.z % p.kv_heads, n0 = blockIdx.y * kPgenRows;
  pdl_launch_dependents();
  pdl_wait();  // nothing of global memory before this: the launch may overlap the kernel ahead
  const int past = static_cast<int>(tree_past(p.past_lengths, 0, b, p.capacity));
  const int tokens = paged_count(pg, b, p.tokens);
  const int end = tokens == 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(past) + tokens, p.capacity));
  const int j0 = static_cast<int>(min(static_cast<int64_t>(blockIdx.x) * p.split_len, static_cast<int64_t>(end)));
  // The last split takes what is left, also past the host's bound.
  const int j1 = static_cast<int>(blockIdx.x + 1 == gridDim.x ? end : min(j0 + p.split_len, static_cast<int64_t>(end)));

  // ---- Q, and where this thread's two rows of scores (g and g + 8) stand.  Over codes Q goes to FP16 by the power of
  // two (2^100 at most) that brings the row's largest element to [2^14, 2^15): 8 bits are exact from 2^-31 of that
  // element on, smaller elements are off by 2^-25 of the scaled row at most (FP16's steps end at 2^-24).
  for (int r = warp; r < kPgenRows; r += kPgenWarps) {
    const int n = n0 + r;
    const uint16_t* src = p.q + ((static_cast<int64_t>(b) * p.tokens + n / group) * p.q_heads + kvh * group + n % group) * D;
    uint32_t x[(D + 63) / 64], top = 0;
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) {
      const int c = 64 * i + 2 * lane;
      x[i] = n < nq && c < D ? __ldg(reinterpret_cast<const uint32_t*>(src + c)) : 0u;
      top = max(top, max(x[i] & 0x7fffu, x[i] >> 16 & 0x7fffu));
    }
    float up = 1.0f;
    if constexpr (kQuant) {
      const int ex = static_cast<int>(__reduce_max_sync(kFull, top) >> 7);
      const int e = ex == 0 || ex == 255 ? 0 : min(14 - (ex - 127), 100);
      up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      if (lane == 0) s_q[r] = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    }
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) {
      const int c = 64 * i + 2 * lane;
      if constexpr (kQuant)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x[i]) : "f"(__uint_as_float(x[i] & 0xffff0000u) * up), "f"(__uint_as_float(x[i] << 16) * up));
      if (c < D) *reinterpret_cast<uint32_t*>(sq + r * kStride + c) = x[i];
    }
  }
  if (threadIdx.x == 0) s_wild = 0;
  int tok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = n0 + g + 8 * h;
    tok[h] = n < nq && n / group < tokens ? n / group : -1;
  }
  const uint8_t* mask = p.mask ? p.mask + b * p.mask_stride : nullptr;
  auto look = [&](int j) {
    if (j >= j1) return -1;
    const int page = paged_page(pg, b, j);
    return page < 0 ? -1 : (page * p.kv_heads + kvh) * pg.page_size + j % pg.page_size;
  };
  if (threadIdx.x < kPgenTile) {
    s_row[0][threadIdx.x] = look(j0 + static_cast<int>(threadIdx.x));
    s_row[1][threadIdx.x] = look(j0 + kPgenTile + static_cast<int>(threadIdx.x));
  }
  __syncthreads();

  // This thread's pieces of a tile: 16 elements of K and of V each.  The next tile's are fetched before this one's
  // arithmetic where registers hold them.
  constexpr int kItems = (kPgenTile * KS + kPgenThreads - 1) / kPgenThreads;
  constexpr bool kAhead = kItems * (FMT == kKvFmtBf16 ? 16 : FMT == kKvFmtE4m3 ? 8 : 6) <= 64;
  PgenRaw<FMT> raw_k[kAhead ? kItems : 1], raw_v[kAhead ? kItems : 1];
  float unit_k = 0.0f, unit_v = 0.0f;  // of key threadIdx.x
  auto fetch = [&](int at) {
    if constexpr (kAhead) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int x = i * kPgenThreads + threadIdx.x, row = x < kPgenTile * KS ? s_row[at][x / KS] : -1;
        raw_k[i] = pgen_fetch16<FMT>(p.k, row, x % KS * 16, D);
        raw_v[i] = pgen_fetch16<FMT>(p.v, row, x % KS * 16, D);
      }
    }
    if (kQuant && threadIdx.x < kPgenTile) {
      const int row = s_row[at][threadIdx.x];
      unit_k = row < 0 ? 0.0f : __ldg(p.k.row_scales + row);
      unit_v = row < 0 ? 0.0f : __ldg(p.v.row_scales + row);
    }
  };
  fetch(0);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, acc[2 * KS][4] = {};
  const float own[2] = {p.scale * (kQuant ? s_q[g] : 1.0f), p.scale * (kQuant ? s_q[g + 8] : 1.0f)};
  int buf = 0;
  for (int base = j0; base < j1; base += kPgenTile) {
    const int next = buf == 2 ? 0 : buf + 1, after = next == 2 ? 0 : next + 1;
    __syncthreads();  // the last tile is read, the next one's rows are there
    const bool drafted = base + kPgenTile > past;
    bool wild = false;
    auto store = [&](int x, const PgenRaw<FMT>& rk, const PgenRaw<FMT>& rv) {
      const int r = x / KS, c = x % KS * 16;
      uint32_t wk[8], wv[8];
      pgen_decode16<FMT>(rk, wk);
      pgen_decode16<FMT>(rv, wv);
      if (drafted && base + r >= past)
#pragma unroll
        for (int e = 0; e < 8; ++e) wild |= pgen_finite<FMT>(wv[e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        *reinterpret_cast<uint4*>(sk + r * kStride + c + 8 * e) =
            make_uint4(wk[4 * e], wk[4 * e + 1], wk[4 * e + 2], wk[4 * e + 3]);
        *reinterpret_cast<uint4*>(sv + r * kStride + c + 8 * e) =
            make_uint4(wv[4 * e], wv[4 * e + 1], wv[4 * e + 2], wv[4 * e + 3]);
      }
    };
    if constexpr (kAhead) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int x = i * kPgenThreads + threadIdx.x;
        if (x < kPgenTile * KS) store(x, raw_k[i], raw_v[i]);
      }
    } else {
#pragma unroll 2
      for (int x = threadIdx.x; x < kPgenTile * KS; x += kPgenThreads) {
        const int row = s_row[buf][x / KS];
        store(x, pgen_fetch16<FMT>(p.k, row, x % KS * 16, D), pgen_fetch16<FMT>(p.v, row, x % KS * 16, D));
      }
    }
    if (kQuant && threadIdx.x < kPgenTile) {
      s_kr[threadIdx.x] = unit_k;
      s_vr[threadIdx.x] = unit_v;
    }
    if (wild) s_wild = 1;
    if (base + kPgenTile < j1) fetch(next);
    if (threadIdx.x < kPgenTile) s_row[after][threadIdx.x] = look(base + 2 * kPgenTile + static_cast<int>(threadIdx.x));
    __syncthreads();
    const int* rows = s_row[buf];
    buf = next;

    const int k0 = warp * 16;
    if (base + k0 >= j1) continue;  // uniform in the warp
    // ---- S: keys k0 + 8 h + 2 tq, + 1
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t a[4], k[4];
      pgen_ldsm4(sq + (lane & 15) * kStride + 16 * ks + 8 * (lane >> 4), a);
      pgen_ldsm4(sk + (k0 + (lane & 7) + 8 * (lane >> 4)) * kStride + 16 * ks + 8 * (lane >> 3 & 1), k);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if constexpr (kQuant)
          asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
              : "+f"(s[h][0]), "+f"(s[h][1]), "+f"(s[h][2]), "+f"(s[h][3])
              : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(k[2 * h]), "r"(k[2 * h + 1]));
        else
          asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
              : "+f"(s[h][0]), "+f"(s[h][1]), "+f"(s[h][2]), "+f"(s[h][3])
              : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(k[2 * h]), "r"(k[2 * h + 1]));
    }
    float top[2] = {-INFINITY, -INFINITY}, unit[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = k0 + 8 * h + 2 * tq + c, j = base + r;
        const bool there = rows[r] >= 0;
        const float k_unit = kQuant ? s_kr[r] : 1.0f;
        unit[h][c] = kQuant ? s_vr[r] : 1.0f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // rows g, g + 8
          float& v = s[h][2 * x + c];
          v = v * own[x] * k_unit;
          const bool sees = there && tok[x] >= 0 &&
                            tree_sees(mask ? mask + static_cast<int64_t>(tok[x]) * p.tokens : nullptr, tok[x], j - past);
          if (!sees) v = -INFINITY;
          top[x] = fmaxf(top[x], v);
        }
      }
    float alpha[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      top[x] = fmaxf(top[x], __shfl_xor_sync(kFull, top[x], 1));
      top[x] = fmaxf(top[x], __shfl_xor_sync(kFull, top[x], 2));
      const float next = fmaxf(m[x], top[x]);
      alpha[x] = m[x] == next || m[x] == -INFINITY ? 1.0f : pgen_exp2((m[x] - next) * 1.44269504f);
      m[x] = next;
      l[x] *= alpha[x];
    }
    if (__any_sync(kFull, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        acc[i][0] *= alpha[0];
        acc[i][1] *= alpha[0];
        acc[i][2] *= alpha[1];
        acc[i][3] *= alpha[1];
      }
    }
    // ---- P, and O: key 2 tq is the k of index tq, 2 tq + 1 that of tq + 4
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t a[4];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float v = s[h][2 * x + c];
          const float w = v == -INFINITY ? 0.0f : pgen_exp2((v - m[x]) * 1.44269504f);
          l[x] += w;
          a[2 * c + x] = v == -INFINITY ? 0u : pgen_tf32(w * unit[h][c]);
        }
      const uint16_t* v0 = sv + (k0 + 8 * h + 2 * tq) * kStride + 2 * g;
#pragma unroll
      for (int i = 0; i < KS; ++i) {  // element 16 i + 2 g in block 2 i, the next in block 2 i + 1
        const float2 x = pgen_pair<FMT>(*reinterpret_cast<const uint32_t*>(v0 + 16 * i));
        const float2 y = pgen_pair<FMT>(*reinterpret_cast<const uint32_t*>(v0 + kStride + 16 * i));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float (&d)[4] = acc[2 * i + e];
          asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
              : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
              : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(__float_as_uint(e ? x.y : x.x)),
                "r"(__float_as_uint(e ? y.y : y.x)));
        }
      }
    }
  }

  // ---- the warps' parts, joined.  acc[2 i + e]: rows g, g + 8, columns 2 tq, 2 tq + 1 of a block: elements 16 i + 2 c + e
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(kFull, l[x], 1);
    l[x] += __shfl_xor_sync(kFull, l[x], 2);
    if (tq == 0) {
      s_m[warp][g + 8 * x] = m[x];
      s_l[warp][g + 8 * x] = l[x];
    }
#pragma unroll
    for (int i = 0; i < KS; ++i)
      *reinterpret_cast<float4*>(so + (warp * kPgenRows + g + 8 * x) * D + 16 * i + 4 * tq) =
          make_float4(acc[2 * i][2 * x], acc[2 * i + 1][2 * x], acc[2 * i][2 * x + 1], acc[2 * i + 1][2 * x + 1]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kPgenRows * D; i += kPgenThreads) {
    const int r = i / D, d = i % D, n = n0 + r;
    if (n >= nq) break;
    const int t = n / group;
    float mx = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kPgenWarps; ++w) mx = fmaxf(mx, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < kPgenWarps; ++w) {
      const float f = s_m[w][r] == -INFINITY ? (s_l[w][r] == 0.0f ? 0.0f : 1.0f) : pgen_exp2((s_m[w][r] - mx) * 1.44269504f);
      sum = fmaf(s_l[w][r], f, sum);
      o = f == 0.0f ? o : fmaf(so[(w * kPgenRows + r) * D + d], f, o);
    }
    if (s_wild && t < tokens) {
      for (int j = max(past, j0); j < j1; ++j) {
        const int row = look(j);
        if (row < 0 || !tree_sees(mask ? mask + static_cast<int64_t>(t) * p.tokens : nullptr, t, j - past)) continue;
        uint32_t w[8];
        pgen_decode16<FMT>(pgen_fetch16<FMT>(p.v, row, d / 16 * 16, D), w);
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 pair = pgen_pair<FMT>(w[e]);
          if (d % 16 / 2 == e) x = d % 2 ? pair.y : pair.x;
        }
        if (!isfinite(x)) o += x;
      }
    }
    const int64_t out = (static_cast<int64_t>(b) * p.tokens + t) * p.q_heads + kvh * group + n % group;
    if (p.splits == 1) {
      p.ctx[out * D + d] = f32_to_bf16_bits(sum == 0.0f ? 0.0f : __fdiv_rn(o, sum));
    } else {
      float* dst = p.partials + (out * p.splits + blockIdx.x) * (D + 2);
      dst[d] = o;
      if (d == 0) {
        dst[D] = mx;
        dst[D + 1] = sum;
      }
    }
  }
}

}  // namespace nvfp4da
