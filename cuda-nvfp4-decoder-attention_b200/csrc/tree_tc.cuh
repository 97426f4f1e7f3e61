// Tree attention for many query rows on the 5th-generation tensor cores
// (head_dim 64 or 128): tcgen05.mma over a BF16, E4M3 or NVFP4 cache.
// Semantics: tree_attention.cuh.  Work line, segments and partials:
// tree_stream.cuh; this kernel replaces the streaming one where a KV head has
// enough query rows to fill 128-row tiles (the rule stands with the launch).
//
// One CTA per SM walks its range of the tile line in segments.  Two streams,
// each a softmax warpgroup with its score buffers, its P tile and its output
// accumulator in tensor memory:
//   up to 128 rows   both streams hold the same rows and take alternate tiles;
//                    their (m, l, o) are joined at the segment's end.  Up to 64
//                    rows, stream 1 sees them in the upper half of its tile, so
//                    that the two streams' live rows sit in all four
//                    tensor-memory quarters (and SM partitions);
//   129 to 256 rows  each stream holds half of the rows and takes every tile.
//
// Roles: warps 0-3 and 4-7 softmax of streams 0 and 1 (one query row per
// thread); warps 8-13 prepare operands; warp 14 issues the MMAs; warp 15 the
// loads.  Per tile of 64 keys:
//   load     codes and scales (TMA, bulk copies) into a ring; BF16 K and V
//            straight into operand tiles;
//   prepare  codes (times the NVFP4 block scale) to FP16, exact, as [key][d]
//            tiles of 128-byte swizzled rows: K is a K-major operand, V an
//            MN-major one, so neither is transposed.  In tiles that reach P_b,
//            V rows past the end and infinities or NaN in V become 0;
//   S = Q K^T   M 128, N 64, into one of the stream's two score buffers;
//   softmax  scores times the row scale of K (FP32), mask, P = 2^(s - m) times
//            the row scale of V over G, to FP16 (BF16 caches: two BF16 terms);
//            the reference m and the scale G move only when passed by a slack
//            of 2^4 and 2^3, and only then the accumulator is rescaled;
//   O += P V  M 128, N = D, accumulated in tensor memory.
// The numerics are those of tree_stream.cuh (P 2^7 p_j gamma_j / G here).
//
// Waits are bounded (one second, shared give-up flag, recorded in
// g_tree_errors); tensor memory is freed on every path.
#pragma once

#include "tree_stream.cuh"

namespace nvfp4da {

constexpr int kTtRows = 128;
constexpr int kTtKeys = 64;
constexpr int kTtSoftmaxWarps = 8;
constexpr int kTtPrepWarps = 6;
constexpr int kTtThreads = (kTtSoftmaxWarps + kTtPrepWarps + 2) * 32;
constexpr int kTtUnitSlots = 8;  // tiles whose row scales are kept
constexpr float kTtPScale = 128.0f;
constexpr float kTtUnitSlack = 8.0f;

template <int D, int FMT, bool SPLIT>  // SPLIT: 129 to 256 rows, half of them per stream
struct TtCfg {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  using Codes = TsCfg<D, FMT, 1, 8>;  // the layout of a ring stage of codes
  static constexpr bool kQuant = FMT != kKvFmtBf16;
  static constexpr int kPanels = D / 64;                      // 64-element panels of a row
  static constexpr uint32_t kOperand = kPanels * kTtKeys * 128;  // a K or V tile, 16-bit
  static constexpr int kK = kQuant ? 2 : 3, kV = SPLIT ? 2 : 3;  // tiles of each in flight
  static constexpr int kStages = kQuant ? (FMT == kKvFmtNvfp4 ? 4 : 3) : 0;  // ring of codes
  static constexpr int kQRows = SPLIT ? 256 : 192;
  static constexpr uint32_t kQPanel = kQRows * 128;
  static constexpr int kTerms = kQuant ? 1 : 2;
  static constexpr uint32_t kP = kTerms * kTtRows * 128;  // per stream
  static constexpr uint32_t kOffK = 0, kOffV = kOffK + kK * kOperand, kOffRing = kOffV + kV * kOperand,
                            kOffQ = kOffRing + kStages * Codes::kStage, kOffP = kOffQ + kPanels * kQPanel,
                            kOffUnits = kOffP + 2 * kP;
  static constexpr uint32_t kUnits = kQuant ? kTtUnitSlots * kTtKeys * 8 : 0;
  static constexpr uint32_t kOffPrefix = kOffUnits + kUnits;
  // The joining area (stream 1's o) overlays Q and P.
  static_assert(kPanels * kQPanel + 2 * kP >= kTtRows * D * 4, "room to join the streams");
  static constexpr uint32_t bytes(int batch) { return kOffPrefix + 8u * (batch + 1) + 1024; }
};

// ---------------------------------------------------------------- tcgen05
// Shared-memory operand descriptors, 128-byte swizzle: start address >> 4
// (bits 0-13), leading (16-29) and stride (32-45) byte offsets >> 4, version 1
// (46), swizzle mode 2 (61-63).  K-major: stride = 1024 between 8-row groups.
// MN-major: stride = 1024 between groups of 8 k, leading = the distance between
// 64-element panels.
__device__ __forceinline__ uint64_t tt_desc(uint32_t saddr, uint32_t leading) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(leading >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// Instruction descriptor, kind::f16: FP32 D, A and B FP16 or BF16, A K-major,
// B K-major or MN-major (bit 16), N >> 3 at 17, M >> 4 at 24.
template <int FMT>
__host__ __device__ constexpr uint32_t tt_idesc(int n, bool mn_major) {
  const uint32_t type = FMT == kKvFmtBf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTtRows >> 4) << 24);
}
__device__ __forceinline__ void tt_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tt_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tt_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tt_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tt_st32(uint32_t taddr, const float (&v)[32]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
      "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
      "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])),
      "r"(__float_as_uint(v[15])), "r"(__float_as_uint(v[16])), "r"(__float_as_uint(v[17])),
      "r"(__float_as_uint(v[18])), "r"(__float_as_uint(v[19])), "r"(__float_as_uint(v[20])),
      "r"(__float_as_uint(v[21])), "r"(__float_as_uint(v[22])), "r"(__float_as_uint(v[23])),
      "r"(__float_as_uint(v[24])), "r"(__float_as_uint(v[25])), "r"(__float_as_uint(v[26])),
      "r"(__float_as_uint(v[27])), "r"(__float_as_uint(v[28])), "r"(__float_as_uint(v[29])),
      "r"(__float_as_uint(v[30])), "r"(__float_as_uint(v[31]))
      : "memory");
}

// Bounded wait; gives up when another role has (`bad`) or after one second.
__device__ __forceinline__ bool tt_wait(uint64_t* bar, uint32_t parity, volatile unsigned* bad) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 0) {
      if (*bad) return false;
      uint64_t t;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (t - t0 > 1000000000ull) {
        atomicOr(&g_tree_errors, static_cast<unsigned>(kErrBarrierTimeout));
        *bad = 1u;
        return false;
      }
    }
  }
}

// (row, 16-byte chunk) of a tile of 128-byte swizzled rows.
__device__ __forceinline__ uint32_t tt_chunk(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

// A counter modulo N with the phase of its mbarriers.
template <int N>
struct TtRing {
  int i = 0;
  uint32_t phase = 0;
  __device__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1u;
    }
  }
};

// Element d of a row of V in global memory, without the row scale.
template <int D, int FMT>
__device__ __forceinline__ float tt_v_global(const KvStore& v, int64_t row, int d) {
  if (FMT == kKvFmtBf16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(v.codes)[row * D + d]);
  if (FMT == kKvFmtE4m3) return f16x2_to_f32x2(e4m3x2_to_f16x2(v.codes[row * D + d])).x;
  const float2 pair = f16x2_to_f32x2(e2m1x2_to_f16x2(v.codes[row * (D / 2) + d / 2]));
  return ((d & 1) ? pair.y : pair.x) * f16x2_to_f32x2(e4m3x2_to_f16x2(v.block_scales[row * (D / 16) + d / 16])).x;
}

template <int D, int FMT, bool SPLIT>
__global__ void __launch_bounds__(kTtThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const TreeStreamParams p) {
  using C = TtCfg<D, FMT, SPLIT>;
  using Codes = typename C::Codes;
  constexpr bool kQuant = C::kQuant;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t ring_full[4], ring_free[4], k_full[3], k_free[3], v_raw[3], v_full[3], v_free[3], q_full,
      s_full[2][2], s_free[2][2], p_full[2], o_done[2], seg_done, join_ready, join_read;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile unsigned s_bad;    // a wait gave up
  __shared__ volatile unsigned s_wild;   // an infinity or NaN was taken out of V
  __shared__ float2 join_ml[kTtRows];
  long long* prefix = reinterpret_cast<long long*>(smem + C::kOffPrefix);
  float2* units_kv = reinterpret_cast<float2*>(smem + C::kOffUnits);  // [slot][key]: row scales of K (scaled) and V

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;
  const int units = p.kv_heads * p.passes;
  const int nq = p.group * p.tokens;

  pdl_launch_dependents();
  if (warp == 14) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&ring_full[i], 1);
      mbar_init(&ring_free[i], kTtPrepWarps);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&k_full[i], kQuant ? kTtPrepWarps : 1);
      mbar_init(&k_free[i], 1);
      mbar_init(&v_raw[i], 1);
      mbar_init(&v_full[i], kTtPrepWarps);
      mbar_init(&v_free[i], 1);
    }
    mbar_init(&q_full, kTtSoftmaxWarps);
    for (int s = 0; s < 2; ++s) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[s][i], 1);
        mbar_init(&s_free[s][i], 4);
      }
      mbar_init(&p_full[s], 4);
      mbar_init(&o_done[s], 1);
    }
    mbar_init(&seg_done, kTtSoftmaxWarps);
    mbar_init(&join_ready, kTtSoftmaxWarps);
    mbar_init(&join_read, 4);
    fence_mbar_init();
    s_bad = 0u;
    s_wild = 0u;
  }
  for (int b = tid; b < p.batch; b += kTtThreads) prefix[b + 1] = (ts_visible(p, b) + kTtKeys - 1) / kTtKeys * units;
  tt_fence_before();
  __syncthreads();
  tt_fence_after();
  if (warp == 0) {
    long long carry = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int b = base + lane;
      long long v = b < p.batch ? prefix[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(kFull, v, o);
        if (lane >= o) v += u;
      }
      if (b < p.batch) prefix[b + 1] = carry + v;
      carry += __shfl_sync(kFull, v, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  const uint32_t tmem = tmem_slot;
  const long long n_tiles = prefix[p.batch];
  const int G = n_tiles < p.grid ? static_cast<int>(n_tiles) : p.grid;
  const long long x0 = cta < G ? n_tiles * cta / G : 0, x1 = cta < G ? n_tiles * (cta + 1) / G : 0;
  TsWalk w;
  bool more = w.begin(prefix, p.batch, units, x0, x1);
  // Tensor memory columns: scores [stream][buffer][64], then o [stream][D].
  auto s_col = [&](int s, int buf) { return tmem + static_cast<uint32_t>((2 * s + buf) * kTtKeys); };
  auto o_col = [&](int s) { return tmem + 256u + static_cast<uint32_t>(s * D); };

  if (warp == 15) {
    // ---------------------------------------------------------------- loads
    if (lane == 0) {
      TtRing<kQuant ? (C::kStages ? C::kStages : 1) : C::kK> rk;
      TtRing<C::kV> rv;
      bool ok = true;
      for (; more && ok; more = w.next()) {
        const int64_t row0 = (static_cast<int64_t>(w.b) * p.kv_heads + w.u / p.passes) * p.capacity;
        for (int t = w.t0; t < w.t1 && ok; ++t) {
          const int64_t row = row0 + static_cast<int64_t>(t) * kTtKeys;
          if constexpr (kQuant) {
            ok = tt_wait(&ring_free[rk.i], rk.phase ^ 1u, &s_bad);
            if (!ok) break;
            uint8_t* st = smem + C::kOffRing + rk.i * Codes::kStage;
            uint64_t* bar = &ring_full[rk.i];
            mbar_arrive_expect_tx(bar, Codes::kTx);
            const int line = static_cast<int>(row * Codes::kRowBytes / 128);
            ts_tma_2d(st, &tm_k, 0, line, bar);
            ts_tma_2d(st + Codes::kOffV, &tm_v, 0, line, bar);
            if constexpr (FMT == kKvFmtNvfp4) {
              bulk_g2s(st + Codes::kOffKb, p.k.block_scales + row * (D / 16), Codes::kBlockScales, bar);
              bulk_g2s(st + Codes::kOffVb, p.v.block_scales + row * (D / 16), Codes::kBlockScales, bar);
            }
            bulk_g2s(st + Codes::kOffKr, p.k.row_scales + row, Codes::kRowScales, bar);
            bulk_g2s(st + Codes::kOffVr, p.v.row_scales + row, Codes::kRowScales, bar);
            rk.next();
          } else {
            ok = tt_wait(&k_free[rk.i], rk.phase ^ 1u, &s_bad);
            if (!ok) break;
            mbar_arrive_expect_tx(&k_full[rk.i], C::kOperand);
            for (int pn = 0; pn < C::kPanels; ++pn)
              ts_tma_2d(smem + C::kOffK + rk.i * C::kOperand + pn * (kTtKeys * 128), &tm_k, pn * 64,
                        static_cast<int>(row), &k_full[rk.i]);
            rk.next();
            ok = tt_wait(&v_free[rv.i], rv.phase ^ 1u, &s_bad);
            if (!ok) break;
            mbar_arrive_expect_tx(&v_raw[rv.i], C::kOperand);
            for (int pn = 0; pn < C::kPanels; ++pn)
              ts_tma_2d(smem + C::kOffV + rv.i * C::kOperand + pn * (kTtKeys * 128), &tm_v, pn * 64,
                        static_cast<int>(row), &v_raw[rv.i]);
            rv.next();
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 14) {
    // ---------------------------------------------------------------- MMAs
    if (lane == 0) {
      constexpr uint32_t kIdescS = tt_idesc<FMT>(kTtKeys, false), kIdescO = tt_idesc<FMT>(D, true);
      TtRing<C::kK> rk;
      TtRing<C::kV> rv;
      uint32_t q_phase = 0, s_count[2] = {0, 0}, p_count[2] = {0, 0};
      bool ok = true;
      for (; more && ok; more = w.next()) {
        const int tiles = w.t1 - w.t0, jobs = SPLIT ? 2 * tiles : tiles;
        const int rows = min(p.rows_per_pass, nq - (w.u % p.passes) * p.rows_per_pass);
        const bool shifted = !SPLIT && rows <= 64;
        ok = tt_wait(&q_full, q_phase, &s_bad);
        q_phase ^= 1u;
        bool begun[2] = {false, false};
        for (int k = 0; k < jobs + 2 && ok; ++k) {
          if (k < jobs) {
            const int s = k & 1, buf = s_count[s] & 1;
            const bool last_use = !SPLIT || s == 1;
            ok = tt_wait(&k_full[rk.i], rk.phase, &s_bad) &&
                 tt_wait(&s_free[s][buf], ((s_count[s] >> 1) & 1) ^ 1u, &s_bad);
            if (!ok) break;
            tt_fence_after();
            // query rows of this stream in the Q tile
            const int q0 = SPLIT ? s * kTtRows : (shifted && s == 0 ? 64 : 0);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t qa = smem_u32(smem + C::kOffQ + (ks >> 2) * C::kQPanel + q0 * 128) + (ks & 3) * 32;
              const uint32_t ka = smem_u32(smem + C::kOffK + rk.i * C::kOperand + (ks >> 2) * (kTtKeys * 128)) + (ks & 3) * 32;
              tt_mma(s_col(s, buf), tt_desc(qa, 16), tt_desc(ka, 16), kIdescS, ks ? 1u : 0u);
            }
            tt_commit(&s_full[s][buf]);
            ++s_count[s];
            if (last_use) {
              tt_commit(&k_free[rk.i]);
              rk.next();
            }
          }
          if (k >= 2) {
            const int s = k & 1;
            const bool last_use = !SPLIT || s == 1;
            ok = tt_wait(&p_full[s], p_count[s] & 1, &s_bad) && tt_wait(&v_full[rv.i], rv.phase, &s_bad);
            if (!ok) break;
            tt_fence_after();
#pragma unroll
            for (int ks = 0; ks < kTtKeys / 16; ++ks) {
              const uint32_t va = smem_u32(smem + C::kOffV + rv.i * C::kOperand) + ks * 2048;
#pragma unroll
              for (int term = 0; term < C::kTerms; ++term) {
                const uint32_t pa = smem_u32(smem + C::kOffP + s * C::kP + term * (kTtRows * 128)) + ks * 32;
                tt_mma(o_col(s), tt_desc(pa, 16), tt_desc(va, kTtKeys * 128), kIdescO,
                       (begun[s] || ks || term) ? 1u : 0u);
              }
            }
            begun[s] = true;
            tt_commit(&o_done[s]);
            ++p_count[s];
            if (last_use) {
              tt_commit(&v_free[rv.i]);
              rv.next();
            }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp >= kTtSoftmaxWarps) {
    // ---------------------------------------------------------------- operands
    const int pt = tid - kTtSoftmaxWarps * 32;  // 0 .. 191
    constexpr int kN = kTtPrepWarps * 32;
    TtRing<C::kStages ? C::kStages : 1> rr;
    TtRing<C::kK> rk;
    TtRing<C::kV> rv;
    int slot = 0;
    bool ok = true;
    for (; more && ok; more = w.next()) {
      const int64_t past = tree_past(p.past_lengths, p.past_length, w.b, p.capacity);
      const int64_t vis = min(past + p.tokens, p.capacity);
      for (int t = w.t0; t < w.t1; ++t) {
        const int64_t key0 = static_cast<int64_t>(t) * kTtKeys;
        const bool edge = key0 + kTtKeys > past;
        const int live = static_cast<int>(min(static_cast<int64_t>(kTtKeys), vis - key0));  // keys before the end
        if constexpr (kQuant) {
          ok = tt_wait(&ring_full[rr.i], rr.phase, &s_bad) && tt_wait(&k_free[rk.i], rk.phase ^ 1u, &s_bad);
          if (!(ok = __all_sync(kFull, ok))) break;
          const uint8_t* st = smem + C::kOffRing + rr.i * Codes::kStage;
          if (pt < kTtKeys) {
            const float kr = reinterpret_cast<const float*>(st + Codes::kOffKr)[pt];
            const float vr = reinterpret_cast<const float*>(st + Codes::kOffVr)[pt];
            units_kv[slot * kTtKeys + pt] = make_float2(kr * p.scale_log2, vr);
          }
          slot = slot + 1 == kTtUnitSlots ? 0 : slot + 1;
          // Items of 16 bytes of codes of one key (NVFP4: 32 elements, E4M3: 16), eight keys side by side.
          constexpr int kItems = Codes::kRowBytes / 16;
          auto prepare = [&](const uint8_t* codes, const uint8_t* blocks, uint8_t* out, bool clean) {
            for (int i = pt; i < kTtKeys * kItems; i += kN) {
              const int c = (i >> 3) % kItems, r = (i / (8 * kItems)) * 8 + (i & 7);
              const uint4 raw = *reinterpret_cast<const uint4*>(codes + ts_swz(r * Codes::kRowBytes + 16 * c));
              const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
              uint32_t h[FMT == kKvFmtNvfp4 ? 16 : 8];
              if constexpr (FMT == kKvFmtNvfp4) {
                const uint32_t two = *reinterpret_cast<const uint16_t*>(blocks + r * (D / 16) + 2 * c);
                const uint32_t b0 = e4m3x2_to_f16x2((two & 0xffu) * 0x101u), b1 = e4m3x2_to_f16x2((two >> 8) * 0x101u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  uint32_t d[4];
                  e2m1x8_to_f16x2x4(word[e], d);
#pragma unroll
                  for (int x = 0; x < 4; ++x) h[4 * e + x] = ts_hmul2(d[x], e < 2 ? b0 : b1);
                }
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) ts_e4m3x4(word[e], h[2 * e], h[2 * e + 1]);
              }
              constexpr int kChunks = FMT == kKvFmtNvfp4 ? 4 : 2;  // 8 elements each
              if (clean) {
                uint32_t bad = 0;
#pragma unroll
                for (int x = 0; x < 4 * kChunks; ++x) h[x] = r < live ? ts_finite<FMT>(h[x], bad) : 0u;
                if (bad) s_wild = 1u;
              }
#pragma unroll
              for (int x = 0; x < kChunks; ++x) {
                const int ch = c * kChunks + x;  // chunk of the whole row
                *reinterpret_cast<uint4*>(out + (ch >> 3) * (kTtKeys * 128) + tt_chunk(r, ch & 7)) =
                    make_uint4(h[4 * x], h[4 * x + 1], h[4 * x + 2], h[4 * x + 3]);
              }
            }
          };
          prepare(st, st + Codes::kOffKb, smem + C::kOffK + rk.i * C::kOperand, false);
          tt_fence_async();
          __syncwarp();
          if (lane == 0) ts_arrive(&k_full[rk.i]);
          rk.next();
          ok = tt_wait(&v_free[rv.i], rv.phase ^ 1u, &s_bad);
          if (!(ok = __all_sync(kFull, ok))) break;
          prepare(st + Codes::kOffV, st + Codes::kOffVb, smem + C::kOffV + rv.i * C::kOperand, edge);
          tt_fence_async();
          __syncwarp();
          if (lane == 0) {
            ts_arrive(&v_full[rv.i]);
            ts_arrive(&ring_free[rr.i]);
          }
          rv.next();
          rr.next();
        } else {
          ok = tt_wait(&v_raw[rv.i], rv.phase, &s_bad);
          if (!(ok = __all_sync(kFull, ok))) break;
          if (edge) {
            uint8_t* v = smem + C::kOffV + rv.i * C::kOperand;
            for (int i = pt; i < kTtKeys * (D / 8); i += kN) {
              const int r = i / (D / 8), ch = i % (D / 8);
              uint4* at = reinterpret_cast<uint4*>(v + (ch >> 3) * (kTtKeys * 128) + tt_chunk(r, ch & 7));
              if (r >= live) {
                *at = make_uint4(0u, 0u, 0u, 0u);
              } else {
                uint32_t bad = 0;
                const uint4 x = *at;
                const uint4 y = make_uint4(ts_finite<FMT>(x.x, bad), ts_finite<FMT>(x.y, bad), ts_finite<FMT>(x.z, bad),
                                           ts_finite<FMT>(x.w, bad));
                if (bad) {
                  *at = y;
                  s_wild = 1u;
                }
              }
            }
            tt_fence_async();
          }
          __syncwarp();
          if (lane == 0) ts_arrive(&v_full[rv.i]);
          rv.next();
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;  // stream, row of its tile
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t s_count = 0, o_phase = 0, end_phase = 0;
    bool first_segment = true;
    int slot0 = 0;  // unit slot of the segment's first tile
    bool ok = true;
    for (; more && ok; more = w.next()) {
      const int b = w.b, kvh = w.u / p.passes, pass = w.u % p.passes, tiles = w.t1 - w.t0;
      const int64_t past = tree_past(p.past_lengths, p.past_length, b, p.capacity);
      const int64_t vis = min(past + p.tokens, p.capacity);
      const int n_first = pass * p.rows_per_pass, rows = min(p.rows_per_pass, nq - n_first);
      const bool shifted = !SPLIT && rows <= 64;
      const int half = (rows + 1) / 2;
      // This thread's query row of the pass (out of [0, rows): none).
      const int n = SPLIT ? (r < half ? s * half + r : rows) : (shifted && s == 1 ? r - 64 : r);
      const bool has = n >= 0 && n < rows;
      const bool warp_has = __any_sync(kFull, has);
      const int tok = has ? (n_first + n) / p.group : 0;
      const int64_t q_row = (static_cast<int64_t>(b) * p.tokens + tok) * p.q_heads +
                            static_cast<int64_t>(kvh) * p.group + (has ? (n_first + n) % p.group : 0);
      if (!SPLIT && s == 1 && !first_segment) {  // stream 0 has read what the join left in the place of Q
        ok = tt_wait(&join_read, end_phase ^ 1u, &s_bad);
        if (!(ok = __all_sync(kFull, ok))) break;
      }
      first_segment = false;
      // ---- Q: this thread's row (SPLIT: all of it; else the panel of its stream)
      float own = kQuant ? 1.0f : p.scale_log2;
      if (has) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + q_row * D);
        float up = 1.0f;
        if constexpr (kQuant) {
          uint32_t top = 0;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 v = __ldg(src + c);
            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) top = max(top, max(e[x] & 0x7fffu, (e[x] >> 16) & 0x7fffu));
          }
          const int ex = static_cast<int>(top >> 7);
          const int e = (ex == 0 || ex == 255) ? 0 : min(14 - (ex - 127), 100);
          up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
          own = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        }
        const int at = SPLIT ? s * kTtRows + r : (shifted ? 64 + n : n);
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          if (!SPLIT && C::kPanels == 2 && (c >> 3) != s) continue;
          if (!SPLIT && C::kPanels == 1 && s == 1) continue;
          uint4 v = __ldg(src + c);
          if constexpr (kQuant) {
            uint32_t* e = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int x = 0; x < 4; ++x)
              e[x] = ts_pack_f16(__uint_as_float(e[x] << 16) * up, __uint_as_float(e[x] & 0xffff0000u) * up);
          }
          *reinterpret_cast<uint4*>(smem + C::kOffQ + (c >> 3) * C::kQPanel + tt_chunk(at, c & 7)) = v;
        }
      }
      tt_fence_async();
      __syncwarp();
      if (lane == 0) ts_arrive(&q_full);

      float m = -INFINITY, l = 0.0f, g_run = kTsMinUnit, p_unit = kTtPScale / kTsMinUnit;
      const uint8_t* mask_row = p.mask ? p.mask + b * p.mask_stride + static_cast<int64_t>(tok) * p.tokens : nullptr;
      uint8_t* pt_base = smem + C::kOffP + s * C::kP;
      int done = 0;  // jobs of this stream in the segment
      for (int i = SPLIT ? 0 : s; i < tiles && ok; i += SPLIT ? 1 : 2, ++done) {
        const int buf = s_count & 1;
        const int64_t key0 = static_cast<int64_t>(w.t0 + i) * kTtKeys;
        ok = tt_wait(&s_full[s][buf], (s_count >> 1) & 1, &s_bad);
        if (!(ok = __all_sync(kFull, ok))) break;
        tt_fence_after();
        ++s_count;
        const float2* unit = units_kv + ((slot0 + i) & (kTtUnitSlots - 1)) * kTtKeys;
        auto tile = [&](auto edge_tag) {
          constexpr bool EDGE = decltype(edge_tag)::value;
          // Keys of the tile this row sees, one bit each.
          unsigned long long seen = ~0ull;
          if constexpr (EDGE) {
            seen = 0;
            for (int e = 0; e < kTtKeys; ++e) {
              const int64_t pos = key0 + e;
              if (has && pos < vis && tree_sees(mask_row, tok, pos - past)) seen |= 1ull << e;
            }
          }
          // ---- maxima: scores (in units of own) and row scales of V
          float mx = -INFINITY;
          [[maybe_unused]] float vx = 0.0f;
          if (warp_has) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[32];
              tt_ld32(s_col(s, buf) + lanes + 32 * h, x);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const bool sees = !EDGE || ((seen >> (32 * h + e)) & 1);
                if constexpr (kQuant) {
                  const float2 uu = unit[32 * h + e];
                  x[e] *= uu.x;
                  if (sees && uu.y < INFINITY) vx = fmaxf(vx, uu.y);
                }
                if (sees) mx = fmaxf(mx, x[e]);
              }
            }
          }
          mx *= own;
          float f = 1.0f;  // what the accumulator is to be scaled by
          if (has && mx > m + kTsSlack) {
            f = m == -INFINITY ? 0.0f : ts_exp2(m - mx);
            l *= f;
            m = mx;
          }
          if constexpr (kQuant) {
            if (has && vx > g_run * kTtUnitSlack) {
              f *= __fdiv_rn(g_run, vx);
              g_run = vx;
              p_unit = __fdiv_rn(kTtPScale, vx);
            }
          }
          // ---- P V of the tile before is done: its P tile is free, its accumulator settled
          if (done > 0) {
            ok = tt_wait(&o_done[s], o_phase, &s_bad);
            o_phase ^= 1u;
            if (!(ok = __all_sync(kFull, ok))) return;
            tt_fence_after();
            if (__any_sync(kFull, f != 1.0f)) {
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                float o[32];
                tt_ld32(o_col(s) + lanes + c, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= f;
                tt_st32(o_col(s) + lanes + c, o);
              }
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
          }
          // ---- P
          if (warp_has) {
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[32];
              tt_ld32(s_col(s, buf) + lanes + 32 * h, x);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                [[maybe_unused]] float2 uu = make_float2(1.0f, 1.0f);
                if constexpr (kQuant) {
                  uu = unit[32 * h + e];
                  x[e] *= uu.x;
                }
                float pj = ts_exp2(fmaf(x[e], own, -m));
                if (EDGE || m == -INFINITY) {
                  const bool sees = !EDGE || ((seen >> (32 * h + e)) & 1);
                  if (!sees || x[e] == -INFINITY) pj = 0.0f;
                  sum += pj;
                  if constexpr (kQuant) pj = sees ? pj * (uu.y * p_unit) : 0.0f;
                } else {
                  sum += pj;
                  if constexpr (kQuant) pj *= uu.y * p_unit;
                }
                x[e] = pj;
              }
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t hi[4];
                [[maybe_unused]] uint32_t lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float a = x[8 * c + 2 * e], d = x[8 * c + 2 * e + 1];
                  if constexpr (kQuant) {
                    hi[e] = ts_pack_f16(a, d);
                  } else {
                    hi[e] = ts_pack_bf16(a, d);
                    lo[e] = ts_pack_bf16(a - __uint_as_float(hi[e] << 16), d - __uint_as_float(hi[e] & 0xffff0000u));
                  }
                }
                uint8_t* at = pt_base + tt_chunk(r, 4 * h + c);
                *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (!kQuant) *reinterpret_cast<uint4*>(at + kTtRows * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            }
            l += sum;
          }
          tt_fence_before();
          tt_fence_async();
          __syncwarp();
          if (lane == 0) {
            ts_arrive(&s_free[s][buf]);
            ts_arrive(&p_full[s]);
          }
        };
        if (key0 + kTtKeys > past) tile(std::true_type{});
        else tile(std::false_type{});
      }
      slot0 = (slot0 + tiles) & (kTtUnitSlots - 1);
      if (ok && done > 0) {
        ok = tt_wait(&o_done[s], o_phase, &s_bad);
        o_phase ^= 1u;
        ok = __all_sync(kFull, ok);
        tt_fence_after();
      }
      // ---- the segment's (m, l, o)
      const float unit_o = kQuant ? g_run * (1.0f / kTtPScale) : 1.0f;
      float4* area = reinterpret_cast<float4*>(smem + C::kOffQ);  // [D / 4][row]
      if (!SPLIT) {
        // Every MMA of the segment has read its Q and P: stream 1 leaves its part in their place.
        __syncwarp();
        if (lane == 0) ts_arrive(&seg_done);
        ok = ok && tt_wait(&seg_done, end_phase, &s_bad);
        ok = __all_sync(kFull, ok);
        if (ok && s == 1 && warp_has) {
          if (done > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tt_ld32(o_col(1) + lanes + c, o);
              if (has)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  area[(c / 4 + e) * kTtRows + n] = make_float4(o[4 * e] * unit_o, o[4 * e + 1] * unit_o,
                                                                o[4 * e + 2] * unit_o, o[4 * e + 3] * unit_o);
            }
          }
          if (has) join_ml[n] = make_float2(m, l);
        }
        tt_fence_before();
        __syncwarp();
        if (lane == 0) ts_arrive(&join_ready);
        ok = ok && tt_wait(&join_ready, end_phase, &s_bad);
        ok = __all_sync(kFull, ok);
        end_phase ^= 1u;
      }
      if (ok && warp_has && (SPLIT || s == 0)) {
        float f0 = unit_o, f1 = 0.0f, mj = m, lj = l;
        if (!SPLIT && tiles > 1) {
          const float2 ml = has ? join_ml[n] : make_float2(-INFINITY, 0.0f);
          mj = fmaxf(m, ml.x);
          const float a0 = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ts_exp2(m - mj);
          f1 = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ts_exp2(ml.x - mj);
          lj = l * a0 + ml.y * f1;
          f0 *= a0;
        }
        const bool whole = w.t0 == 0 && w.t1 == w.nt;
        const int64_t slot = 2 * static_cast<int64_t>(cta) + (w.x == x0 ? 0 : 1);
        const float inv = lj == 0.0f ? 0.0f : __fdiv_rn(1.0f, lj);
        const int64_t v_row = (static_cast<int64_t>(b) * p.kv_heads + kvh) * p.capacity;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tt_ld32(o_col(s) + lanes + c, o);
          if (!has) continue;  // tt_ld32 brings the lanes together again
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = f0 == 0.0f ? 0.0f : o[e] * f0;
          if (f1 != 0.0f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 x = area[(c / 4 + e) * kTtRows + n];
              o[4 * e] = fmaf(x.x, f1, o[4 * e]);
              o[4 * e + 1] = fmaf(x.y, f1, o[4 * e + 1]);
              o[4 * e + 2] = fmaf(x.z, f1, o[4 * e + 2]);
              o[4 * e + 3] = fmaf(x.w, f1, o[4 * e + 3]);
            }
          }
          if (s_wild) {  // infinities and NaN of V that were taken out, for the rows that see them
            const int64_t first = max(past, static_cast<int64_t>(w.t0) * kTtKeys);
            const int64_t last = min(vis, static_cast<int64_t>(w.t1) * kTtKeys);
            for (int64_t pos = first; pos < last; ++pos) {
              if (!tree_sees(mask_row, tok, pos - past)) continue;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float x = tt_v_global<D, FMT>(p.v, v_row + pos, c + e);
                if (!isfinite(x)) o[e] += x;
              }
            }
          }
          if (whole) {
            uint4* dst = reinterpret_cast<uint4*>(p.ctx + q_row * D + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t x[4];
#pragma unroll
              for (int y = 0; y < 4; ++y)
                x[y] = lj == 0.0f ? 0u : ts_pack_bf16(o[8 * e + 2 * y] * inv, o[8 * e + 2 * y + 1] * inv);
              dst[e] = make_uint4(x[0], x[1], x[2], x[3]);
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(p.part_o + (slot * p.rows_per_pass + n) * D + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (has && !whole) p.part_ml[slot * p.rows_per_pass + n] = make_float2(mj, lj);
      }
      tt_fence_before();
      __syncwarp();
      if (!SPLIT && s == 0 && lane == 0) ts_arrive(&join_read);
    }
  }
  tt_fence_before();
  __syncthreads();
  if (warp == 14) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace nvfp4da
