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
// thread); warps 8-11 prepare K and 12-15 V; warps 16 and 18 issue the MMAs of
// a stream each (one warp for both could not issue them fast enough beside the
// others on its scheduler); warp 17 loads codes, warp 19 scales.  Per tile of 64
// keys:
//   load     codes (TMA) and scales (16-byte asynchronous copies) into a ring;
//            BF16 K and V straight into operand tiles;
//   prepare  codes (times the NVFP4 block scale) to FP16, exact, as [key][d]
//            tiles of 128-byte swizzled rows: K is a K-major operand, V an
//            MN-major one, so neither is transposed.  In tiles that reach P_b,
//            V rows past the end and infinities or NaN in V become 0;
//   S = Q K^T   M 128, N 64, into one of the stream's two score buffers;
//   softmax  scores times the row scale of K (FP32), mask, P = 2^(s - m) times
//            the row scale of V, to FP16 (BF16 caches: two BF16 terms), written
//            over the scores in tensor memory; the reference m moves only when
//            P would pass 2^15 (BF16: when a score passes m by 2^20), and only
//            then the accumulator is rescaled;
//   O += P V  M 128, N = D, P read from tensor memory, accumulated there over the
//            segment.  The tensor cores' sums round down: 131,008 equal values in
//            one segment (D 64) come out low by 2^-13, 1/16 of BF16's half step.
// Shared memory feeds the MMAs, so P stays out of it: with P as a
// shared-memory operand its reads and writes took a third of the bandwidth and
// the kernel 1.6 times as long.
// The numerics are those of tree_stream.cuh, but that over codes m serves the
// weights and the contributions 2^(s - m) gamma_j alike: it is set by the largest
// contribution, which comes to 2^4 to 2^6.
//
// What bounds it, at 1.9 GHz.  Over codes with up to 128 rows: the roles' own
// latency.  A tile's MMAs take 650 cycles (49 for a step of K Q^T, read from
// shared memory, 65 for one of P V), but a softmax warp, alone on its scheduler
// but for two preparing warps, takes 1,450 a tile of its stream, and preparing
// one 1,400; the pipeline moves a tile every 1,400.  16 tokens over NVFP4 (8
// sequences x 6 heads, 30,001 to 32,752 positions): 155 to 157 us, 316 TFLOP/s,
// tensor pipe 32 % busy; where the compiler puts the rarely run code moves that by
// up to 14 %.  Over BF16 with more than 128 rows: the MMAs, since P is two
// terms: 1,824 of some 2,400 cycles a tile of 256 rows, 75 % of them rows.  48
// tokens (16 sequences, 8,000 positions): 130 to 137 us on several machines, 416
// to 438 TFLOP/s, pipe 56 % busy.
// A segment costs 15,000 to 20,000 cycles beside its tiles: the walk, Q, the
// first tile's second pass, the join and the partial results.
// Tried, and not kept: the two preparing groups taking K and V of alternate tiles
// (every ring then needs an even number of buffers; 165 -> 170 us), scores and
// P V issued in whatever order they are ready (-> 176 us), more buffers for K
// and V, three shares of registers.
//
// Waits are bounded as in tree_stream.cuh; a CTA that gives up lets its copies
// and MMAs in flight end (or a further limit pass), and frees its tensor memory.
#pragma once

#include "tree_stream.cuh"

namespace nvfp4da {

constexpr int kTtRows = 128;
constexpr int kTtKeys = 64;
constexpr int kTtSoftmaxWarps = 8;
constexpr int kTtPrepWarps = 8;
constexpr int kTtMmaWarp = kTtSoftmaxWarps + kTtPrepWarps, kTtLoadWarp = kTtMmaWarp + 1;
constexpr int kTtThreads = (kTtSoftmaxWarps + kTtPrepWarps + 4) * 32;  // whole warpgroups
// Registers: 96 a thread at launch (640 threads); the softmax warps take what
// the others give: 256 * 144 + 384 * 64 = 640 * 96.
constexpr int kTtSoftmaxRegs = 144, kTtOtherRegs = 64;
constexpr int kTtUnitSlots = 8;  // tiles whose row scales are kept
// Over codes P = 2^(s - m) gamma_j, in FP16, has one reference m for both the softmax and the contributions: the
// largest contribution that m is set by comes to 2^4 to 2^6, a later one may be up to 2^15.  A weight 2^(s - m)
// itself is at most 2^kTtHead when m is set, so that rows of V that are all tiny leave l in range.
constexpr float kTtTop = 5.0f, kTtHead = 100.0f;
constexpr float kTtSumLimit = 1.32922800e+36f, kTtSumStep = 32.0f;  // 2^120: m moves up by 32 where l would pass it

template <int D, int FMT, bool SPLIT>  // SPLIT: 129 to 256 rows, half of them per stream
struct TtCfg {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  using Codes = TsCfg<D, FMT, 1, 8, 1, 64>;  // the layout of a ring stage of codes
  static constexpr bool kQuant = FMT != kKvFmtBf16;
  static constexpr int kPanels = D / 64;                      // 64-element panels of a row
  static constexpr uint32_t kOperand = kPanels * kTtKeys * 128;  // a K or V tile, 16-bit
  static constexpr int kK = kQuant ? (SPLIT ? 2 : 3) : 4;  // K and V tiles in flight
  static constexpr int kV = kQuant ? 3 : 4;
  static constexpr int kStages = kQuant ? (FMT == kKvFmtNvfp4 ? 4 : 3) : 0;  // ring of codes
  static constexpr int kQRows = SPLIT ? 256 : 192;
  static constexpr uint32_t kQPanel = kQRows * 128;
  static constexpr uint32_t kOffK = 0, kOffV = kOffK + kK * kOperand, kOffRing = kOffV + kV * kOperand,
                            kOffQ = kOffRing + kStages * Codes::kStage, kOffUnits = kOffQ + kPanels * kQPanel;
  // Row scales of a tile's keys: K (times log2(e) / sqrt(D)), V.
  static constexpr uint32_t kUnitFloats = 2 * kTtKeys;
  static constexpr uint32_t kUnits = kQuant ? kTtUnitSlots * kUnitFloats * 4 : 0;
  static constexpr uint32_t kOffPrefix = kOffUnits + kUnits;
  // Stream 1's o of up to 64 rows overlays Q when the streams are joined.
  static_assert(kPanels * kQPanel >= 64u * D * 4, "room to join the streams");
  template <bool PAGED = false>
  static constexpr uint32_t bytes(int batch) { return kOffPrefix + (PAGED ? 12u : 4u) * (batch + 1) + 1024; }
};

// PAGED: what a segment costs beside its tiles, in tiles (see kTsSegment).  us for 0, 4, 8, 12, 16 of them: 64 rows of 32
// sequences of 100 to 4,000 positions, head_dim 128, BF16 91, 56, 52, 52, 52, NVFP4 120, 75, 64, 61, 62.
constexpr int kTtSegment = 12;
constexpr int kTtGoneSlots = 16;  // tiles whose missing pages are kept: more than the loads are ahead of the softmax

// ---------------------------------------------------------------- tcgen05
// Shared-memory operand descriptors, 128-byte swizzle: start address >> 4
// (bits 0-13), leading (16-29) and stride (32-45) byte offsets >> 4, version 1
// (46), swizzle mode 2 (61-63).  K-major: stride = 1024 between 8-row groups.
// MN-major: stride = 1024 between groups of 8 k, leading = the distance between
// 64-element panels.
// Only the start address varies: the low words are added up in 32 bits.
constexpr uint32_t kTtDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tt_desc_low(uint32_t saddr, uint32_t leading) {
  return ((saddr & 0x3FFFFu) >> 4) | ((leading >> 4) << 16);
}
// Instruction descriptor, kind::f16: FP32 D, A and B FP16 or BF16, A K-major,
// B K-major or MN-major (bit 16), N >> 3 at 17, M >> 4 at 24.
template <int FMT>
__host__ __device__ constexpr uint32_t tt_idesc(int n, bool mn_major) {
  const uint32_t type = FMT == kKvFmtBf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTtRows >> 4) << 24);
}
__device__ __forceinline__ void tt_mma(uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %5, 0;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}" ::"r"(tmem_d),
      "r"(a_low), "r"(b_low), "r"(kTtDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in tensor memory.
__device__ __forceinline__ void tt_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_low, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n mov.b64 b, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_low), "r"(kTtDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One lane of the (converged) warp.
__device__ __forceinline__ bool tt_elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tt_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tt_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 32 columns of this warp's lanes, without waiting for them.
__device__ __forceinline__ void tt_ld32_async(uint32_t taddr, float* v) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// After tt_wait_ld: nothing may use v[0 .. N) earlier.
template <int N>
__device__ __forceinline__ void tt_loaded(float* v) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tt_ld32(uint32_t taddr, float (&v)[32]) {
  tt_ld32_async(taddr, v);
  tt_wait_ld();
  tt_loaded<32>(v);
}
__device__ __forceinline__ void tt_ld16(uint32_t taddr, float (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr));
  tt_wait_ld();
  tt_loaded<16>(v);
}
__device__ __forceinline__ void tt_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// Column of P, in its score buffer, of the MMA step of keys 16 ks ..: FP16
// pairs, or per 32 keys the first BF16 terms and then the second (the scores of
// the other 32 keys stay whole until they are read).
template <int FMT>
__host__ __device__ constexpr uint32_t tt_p_col(int ks) {
  return FMT == kKvFmtBf16 ? (ks >> 1) * 32 + (ks & 1) * 8 : ks * 8;
}
// Two FP32 operations in one instruction.
__device__ __forceinline__ float2 tt_mul2(float2 a, float2 b) {
  float2 c;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n"
      " mov.b64 {%0, %1}, z;\n}" : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ float2 tt_add2(float2 a, float2 b) {
  float2 c;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n"
      " mov.b64 {%0, %1}, z;\n}" : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ float2 tt_fma2(float2 a, float2 b, float2 d) {
  float2 c;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 w, {%6, %7};\n"
      " fma.rn.f32x2 z, x, y, w;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(d.x), "f"(d.y));
  return c;
}

// (row, 16-byte chunk) of a tile of 128-byte swizzled rows.
__device__ __forceinline__ uint32_t tt_chunk(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

// The whole part of log2 |x| (-127 below 2^-126), -inf where x is not finite.
__device__ __forceinline__ float tt_log2(float x) {
  const uint32_t e = __float_as_uint(x) >> 23 & 0xffu;
  return e == 255u ? -INFINITY : __uint_as_float(0x4b000000u | e) - 8388735.0f;  // 2^23 + e, less 2^23 + 127
}

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

// PAGED: a tile's boxes come from the pages that the block table names, K's by the loading warp and V's by the one
// that copies scales; boxes of pages that are not there, and their scales, come in as zeros, and the softmax leaves
// their keys out.
template <int D, int FMT, bool SPLIT, bool PAGED = false>
__global__ void __launch_bounds__(kTtThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const TreeStreamParams p) {
  using C = TtCfg<D, FMT, SPLIT>;
  using Codes = typename C::Codes;
  constexpr bool kQuant = C::kQuant;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // Pointer arithmetic, not an integer round trip: the compiler then knows that
  // what it points to is shared memory.
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t ring_full[4], ring_free[4], k_full[4], k_free[4], v_raw[4], v_full[4], v_free[4], q_full,
      s_full[2][2], p_full[2][2], o_done[2], o_end[2], seg_done, join_ready, join_read, drained[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile unsigned s_bad;    // a wait gave up
  __shared__ volatile unsigned s_wild;   // an infinity or NaN was taken out of V
  [[maybe_unused]] __shared__ unsigned s_gone[PAGED ? kTtGoneSlots : 1];  // of a tile, 16-key slices that are not there
  [[maybe_unused]] __shared__ int s_range[PAGED ? 4 : 1];                 // places, G, first tile, end
  __shared__ float4 join[2][kTtRows];    // a stream's m, l and the unit of its o, where the two are joined
  int* prefix = reinterpret_cast<int*>(smem + C::kOffPrefix);
  float* units_kv = reinterpret_cast<float*>(smem + C::kOffUnits);  // [slot][kUnitFloats]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;
  const int units = p.kv_heads * p.passes;
  const int nq = p.group * p.tokens;

  pdl_launch_dependents();
  if (warp == kTtMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&ring_full[i], PAGED ? 34 : 33);  // the codes' bytes, and the lanes that copy scales
      mbar_init(&ring_free[i], kTtPrepWarps);
      mbar_init(&k_full[i], kQuant ? kTtPrepWarps / 2 : 1);
      mbar_init(&k_free[i], SPLIT ? 2 : 1);  // each stream that reads the tile
      mbar_init(&v_raw[i], 1);
      mbar_init(&v_full[i], kTtPrepWarps / 2);
      mbar_init(&v_free[i], SPLIT ? 2 : 1);
    }
    const uint32_t active = ((SPLIT ? (p.rows_per_pass + 1) / 2 : p.rows_per_pass) + 31) / 32;  // softmax warps
    mbar_init(&q_full, 2 * active);
    for (int s = 0; s < 2; ++s) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[s][i], 1);
        mbar_init(&p_full[s][i], active);  // per buffer: a warp may be one job ahead of another
      }
      mbar_init(&o_done[s], 1);
      mbar_init(&o_end[s], 1);
      mbar_init(&drained[s], 1);
    }
    mbar_init(&seg_done, 2 * active);
    mbar_init(&join_ready, 2 * active);
    mbar_init(&join_read, 2 * active);
    fence_mbar_init();
    s_bad = 0u;
    s_wild = 0u;
  }
  // Nothing of global memory before this: the launch may overlap the kernel ahead.
  pdl_wait();
  if (tid < 2) p.part_slots[2 * cta + tid] = make_int4(-1, 0, 0, 0);
  tt_fence_before();
  ts_prefix<PAGED>(p, units, kTtKeys, prefix);
  if constexpr (PAGED) {
    if (tid == 0) {
      const int places = ts_places(p, prefix, units), g = min(places, p.grid);
      s_range[0] = places;
      s_range[1] = g;
      s_range[2] = cta < g ? ts_first_tile_weighted(p, prefix, units, cta, g) : 0;
      s_range[3] = cta < g ? ts_first_tile_weighted(p, prefix, units, cta + 1, g) : 0;
    }
    __syncthreads();
  }
  tt_fence_after();
  const uint32_t tmem = tmem_slot;
  // Tensor memory columns: scores [stream][buffer][64], then o [stream][D].
  auto s_col = [&](int s, int buf) { return tmem + static_cast<uint32_t>((2 * s + buf) * kTtKeys); };
  auto o_col = [&](int s) { return tmem + 256u + static_cast<uint32_t>(s * D); };

  // Each role walks the CTA's range itself (kept apart, so that no role holds
  // another's registers).
  auto range = [&](int& n_tiles, int& G, int& x0) {
    if constexpr (PAGED) {
      n_tiles = s_range[0];
      G = s_range[1];
      x0 = s_range[2];
      return s_range[3];
    }
    n_tiles = prefix[p.batch];
    G = min(n_tiles, p.grid);
    x0 = cta < G ? ts_first_tile(n_tiles, cta, G) : 0;
    return cta < G ? ts_first_tile(n_tiles, cta + 1, G) : 0;
  };
  // Softmax warps of a stream that hold rows (the others leave at once): those
  // of the first `active` quarters of a tile, or, where stream 1 sees up to 64
  // rows in the upper half, from its third on.
  const bool upper = !SPLIT && p.rows_per_pass <= 64;
  const int active = ((SPLIT ? (p.rows_per_pass + 1) / 2 : p.rows_per_pass) + 31) / 32;
  auto begin = [&](TsWalk& w) {
    int n_tiles, G, x0;
    const int x1 = range(n_tiles, G, x0);
    return w.begin(prefix, p.batch, units, x0, x1);
  };

  if (warp >= kTtSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTtOtherRegs));
    TsWalk w;
    bool more = begin(w);
    if (PAGED && (warp == kTtLoadWarp || warp == kTtLoadWarp + 2)) {
      // ---------------------------------------------------------------- pages: K, or V and the scales of both
      const bool is_v = warp != kTtLoadWarp;
      constexpr int kRing = kQuant ? (C::kStages ? C::kStages : 1) : C::kK;
      static_assert(kQuant || C::kK == C::kV, "one ring each of the same length");
      uint64_t* full = kQuant ? ring_full : is_v ? v_raw : k_full;
      uint64_t* empty = kQuant ? ring_free : is_v ? v_free : k_free;
      TsBoxes<kTtKeys> at;
      TtRing<kRing> r;
      int filled = 0;
      bool ok = true;
      for (; more && ok; more = w.next()) {
        at.begin(p, w.b, w.u / p.passes, ts_lengths(p, prefix)[w.b].y, w.t0, w.t1, lane);
        for (int t = w.t0; t < w.t1; ++t) {
          ok = __all_sync(kFull, ts_wait(&empty[r.i], r.phase ^ 1u, &s_bad));
          if (!ok) break;
          at.advance(p, t, lane);
          const int mine = at.row(t, lane << p.box_log2), of_slice = at.row(t, lane * 16);
          const unsigned gone = __ballot_sync(kFull, lane < kTtKeys / 16 && of_slice < 0);
          if (lane == 0) {
            if (!is_v) s_gone[filled & (kTtGoneSlots - 1)] = gone;
            mbar_arrive_expect_tx(&full[r.i], kQuant ? Codes::kCodes : C::kOperand);
          }
          __syncwarp();
          uint8_t* st = smem + (kQuant ? C::kOffRing + r.i * Codes::kStage
                                       : (is_v ? C::kOffV : C::kOffK) + r.i * C::kOperand);
          if (lane < 1 << at.per_log2) {
            // Behind the pool's last row: zeros.
            const int from = mine >= 0 ? mine : p.pg.pages * p.kv_heads * p.pg.page_size;
            const CUtensorMap* map = is_v ? &tm_v : &tm_k;
            if constexpr (kQuant) {  // rows stand in groups of 16
              ts_tma_2d(st + (is_v ? Codes::kOffV : 0) + (lane << p.box_log2) * Codes::kRowBytes, map, 0,
                        from / 16 * (16 * Codes::kRowBytes / 128), &full[r.i]);
            } else {
#pragma unroll
              for (int pn = 0; pn < C::kPanels; ++pn)
                ts_tma_2d(st + pn * (kTtKeys * 128) + (lane << p.box_log2) * 128, map, pn * 64, from, &full[r.i]);
            }
          }
          __syncwarp();
          if constexpr (kQuant) {
            if (is_v) {
              ts_load_scales_paged<D, FMT, Codes, kTtKeys>(st + Codes::kOffKb, st + Codes::kOffKr, p.k, at, t, lane);
              ts_load_scales_paged<D, FMT, Codes, kTtKeys>(st + Codes::kOffVb, st + Codes::kOffVr, p.v, at, t, lane);
              ts_copy_arrive(&full[r.i]);
            }
          }
          ++filled;
          r.next();
        }
      }
      if constexpr (kQuant) ts_copies_landed();
      if (lane == 0) ts_all_landed<kRing>(full, filled);
      __syncwarp();
    } else if (kQuant && warp == kTtLoadWarp + 2) {
      // ---------------------------------------------------------------- scales (see ts_load_scales)
      const int64_t all_rows = static_cast<int64_t>(p.batch) * p.kv_heads * p.capacity;
      TtRing<C::kStages ? C::kStages : 1> rk;
      bool ok = true;
      for (; more && ok; more = w.next()) {
        const int64_t row0 = (static_cast<int64_t>(w.b) * p.kv_heads + w.u / p.passes) * p.capacity;
        for (int t = w.t0; t < w.t1; ++t) {
          ok = __all_sync(kFull, ts_wait(&ring_free[rk.i], rk.phase ^ 1u, &s_bad));
          if (!ok) break;
          uint8_t* st = smem + C::kOffRing + rk.i * Codes::kStage;
          ts_load_scales<D, FMT, Codes, kTtKeys>(st, p, row0 + t * kTtKeys, all_rows, lane);
          ts_copy_arrive(&ring_full[rk.i]);
          rk.next();
        }
      }
      ts_copies_landed();
    } else if (warp == kTtLoadWarp) {
      // ---------------------------------------------------------------- loads
      if (lane == 0) {
        TtRing<kQuant ? (C::kStages ? C::kStages : 1) : C::kK> rk;
        TtRing<C::kV> rv;
        int filled = 0, filled_v = 0;  // codes or K, V
        bool ok = true;
        for (; more && ok; more = w.next()) {
          const int64_t row0 = (static_cast<int64_t>(w.b) * p.kv_heads + w.u / p.passes) * p.capacity;
          for (int t = w.t0; t < w.t1 && ok; ++t) {
            const int64_t row = row0 + t * kTtKeys;
            if constexpr (kQuant) {
              ok = ts_wait(&ring_free[rk.i], rk.phase ^ 1u, &s_bad);
              if (!ok) break;
              uint8_t* st = smem + C::kOffRing + rk.i * Codes::kStage;
              uint64_t* bar = &ring_full[rk.i];
              mbar_arrive_expect_tx(bar, 2 * Codes::kCodes);
              const int line = static_cast<int>(row * Codes::kRowBytes / 128);
              ts_tma_2d(st, &tm_k, 0, line, bar);
              ts_tma_2d(st + Codes::kOffV, &tm_v, 0, line, bar);
              ++filled;
              rk.next();
            } else {
              ok = ts_wait(&k_free[rk.i], rk.phase ^ 1u, &s_bad);
              if (!ok) break;
              mbar_arrive_expect_tx(&k_full[rk.i], C::kOperand);
              for (int pn = 0; pn < C::kPanels; ++pn)
                ts_tma_2d(smem + C::kOffK + rk.i * C::kOperand + pn * (kTtKeys * 128), &tm_k, pn * 64,
                          static_cast<int>(row), &k_full[rk.i]);
              ++filled;
              rk.next();
              ok = ts_wait(&v_free[rv.i], rv.phase ^ 1u, &s_bad);
              if (!ok) break;
              mbar_arrive_expect_tx(&v_raw[rv.i], C::kOperand);
              for (int pn = 0; pn < C::kPanels; ++pn)
                ts_tma_2d(smem + C::kOffV + rv.i * C::kOperand + pn * (kTtKeys * 128), &tm_v, pn * 64,
                          static_cast<int>(row), &v_raw[rv.i]);
              ++filled_v;
              rv.next();
            }
          }
        }
        if constexpr (kQuant) {
          ts_all_landed<C::kStages ? C::kStages : 1>(ring_full, filled);
        } else {
          ts_all_landed<C::kK>(k_full, filled);
          ts_all_landed<C::kV>(v_raw, filled_v);
        }
      }
      __syncwarp();
    } else if (warp == kTtMmaWarp || warp == kTtMmaWarp + 2) {
      // ---------------------------------------------------------------- MMAs, a warp per stream
      // The whole warp walks the line, one lane issues.  The stream's P takes the
      // place of its scores: the scores of job n + 2 go into the buffer that held
      // P of job n, after that job's P V in issue order.
      constexpr uint32_t kIdescS = tt_idesc<FMT>(kTtKeys, false), kIdescO = tt_idesc<FMT>(D, true);
      const int s = (warp - kTtMmaWarp) / 2;
      const bool issuer = tt_elect();
      const uint32_t base = smem_u32(smem), o_at = o_col(s);
      TtRing<C::kK> rk;
      TtRing<C::kV> rv;
      uint32_t q_phase = 0, nth = 0, nth_s = 0;  // P V and scores issued, over all segments
      bool ok = true;
      for (; more && ok; more = w.next()) {
        const int tiles = w.t1 - w.t0;
        const int rows = min(p.rows_per_pass, nq - (w.u % p.passes) * p.rows_per_pass);
        const bool shifted = upper;
        // query rows of this stream in the Q tile
        const uint32_t q0 = SPLIT ? s * kTtRows : (shifted && s == 0 ? 64 : 0);
        const uint32_t qa = tt_desc_low(base + C::kOffQ + q0 * 128, 16);
        ok = __all_sync(kFull, ts_wait(&q_full, q_phase, &s_bad));
        q_phase ^= 1u;
        auto scores = [&] {
          ok = __all_sync(kFull, ts_wait(&k_full[rk.i], rk.phase, &s_bad));
          if (!ok) return;
          tt_fence_after();
          const uint32_t ka = tt_desc_low(base + C::kOffK + rk.i * C::kOperand, 16);
          const uint32_t d = s_col(s, nth_s & 1);
          if (issuer) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              tt_mma(d, qa + ((ks >> 2) * C::kQPanel + (ks & 3) * 32) / 16,
                     ka + ((ks >> 2) * (kTtKeys * 128) + (ks & 3) * 32) / 16, kIdescS, ks ? 1u : 0u);
            tt_commit(&s_full[s][nth_s & 1]);
            tt_commit(&k_free[rk.i]);
          }
          __syncwarp();
          ++nth_s;
        };
        // Tiles in order; without SPLIT every other one is this stream's.
        int next_s = 0;  // tile whose scores come next
        auto advance_scores = [&] {
          while (next_s < tiles) {
            const bool mine = SPLIT || (next_s & 1) == s;
            if (mine) scores();
            rk.next();
            ++next_s;
            if (mine) break;
          }
        };
        advance_scores();
        if (ok) advance_scores();
        for (int t = 0; t < tiles && ok; ++t) {
          if (SPLIT || (t & 1) == s) {
            ok = ts_wait(&p_full[s][nth & 1], (nth >> 1) & 1, &s_bad) && ts_wait(&v_full[rv.i], rv.phase, &s_bad);
            if (!(ok = __all_sync(kFull, ok))) break;
            tt_fence_after();
            const uint32_t va = tt_desc_low(base + C::kOffV + rv.i * C::kOperand, kTtKeys * 128);
            const uint32_t pa = s_col(s, nth & 1);
            const uint32_t begun = t >= (SPLIT ? 1 : 2) ? 1u : 0u;  // not the stream's first tile of the segment
            if (issuer) {
#pragma unroll
              for (int ks = 0; ks < kTtKeys / 16; ++ks) {
                tt_mma_ts(o_at, pa + tt_p_col<FMT>(ks), va + ks * 2048 / 16, kIdescO, ks ? 1u : begun);
                if constexpr (!kQuant) tt_mma_ts(o_at, pa + tt_p_col<FMT>(ks) + 16, va + ks * 2048 / 16, kIdescO, 1u);
              }
              tt_commit(&o_done[s]);
              tt_commit(&v_free[rv.i]);
            }
            __syncwarp();
            ++nth;
            advance_scores();
          }
          rv.next();
        }
        while (next_s < tiles) {  // the other stream's last tile
          rk.next();
          ++next_s;
        }
        if (ok && issuer) tt_commit(&o_end[s]);
        __syncwarp();
      }
    } else if (warp >= kTtSoftmaxWarps && warp < kTtMmaWarp) {
      // ---------------------------------------------------------------- operands: warps 8-11 K, 12-15 V
      const bool is_v = warp >= kTtSoftmaxWarps + kTtPrepWarps / 2;
      constexpr int kN = kTtPrepWarps / 2 * 32;
      const int pt = (tid - kTtSoftmaxWarps * 32) % kN;
      // Items of 16 bytes of codes of one key (NVFP4: 32 elements, E4M3: 16),
      // eight keys side by side; a thread's items of a tile are kStep keys apart
      // (a multiple of 8: the same swizzle), or, D = 64, all in one row.
      constexpr int kItems = kQuant ? Codes::kRowBytes / 16 : 1;
      constexpr int kRounds = (kTtKeys * kItems + kN - 1) / kN, kStep = kN / kItems;
      constexpr int kChunks = FMT == kKvFmtNvfp4 ? 4 : 2;  // 16-byte chunks of 8 elements an item becomes
      const int c0 = (pt >> 3) % kItems, r0 = (pt / (8 * kItems)) * 8 + (pt & 7);
      const bool busy = r0 < kTtKeys;
      const uint32_t src0 = (is_v ? Codes::kOffV : 0u) + ts_swz(r0 * Codes::kRowBytes + 16 * c0);
      const uint32_t scale0 = (is_v ? Codes::kOffVb : Codes::kOffKb) + r0 * (D / 16) + 2 * c0;
      uint32_t dst0[kChunks];
#pragma unroll
      for (int y = 0; y < kChunks; ++y) {
        const int ch = c0 * kChunks + y;  // chunk of the whole row
        dst0[y] = (ch >> 3) * (kTtKeys * 128) + tt_chunk(r0, ch & 7);
      }
      TtRing<C::kStages ? C::kStages : 1> rr;
      TtRing<C::kK> rk;
      TtRing<C::kV> rv;
      int slot = 0;
      bool ok = true;
      for (; more && ok; more = w.next()) {
        const int past = PAGED ? ts_lengths(p, prefix)[w.b].x : ts_past(p, w.b);
        const int vis = PAGED ? ts_lengths(p, prefix)[w.b].y : ts_visible(p, w.b);
        for (int t = w.t0; t < w.t1; ++t) {
          const int key0 = t * kTtKeys;
          const bool edge = key0 + kTtKeys > past;
          const int live = min(kTtKeys, vis - key0);  // keys before the end
          if constexpr (kQuant) {
            ok = ts_wait(&ring_full[rr.i], rr.phase, &s_bad);
            if (!(ok = __all_sync(kFull, ok))) break;
            const uint8_t* st = smem + C::kOffRing + rr.i * Codes::kStage;
            uint4 raw[kRounds];
            [[maybe_unused]] uint32_t scales[kRounds];
            if (busy) {
#pragma unroll
              for (int x = 0; x < kRounds; ++x) {
                raw[x] = *reinterpret_cast<const uint4*>(st + src0 + x * kStep * Codes::kRowBytes);
                if constexpr (FMT == kKvFmtNvfp4)
                  scales[x] = *reinterpret_cast<const uint16_t*>(st + scale0 + x * kStep * (D / 16));
              }
            }
            [[maybe_unused]] float2 kr, vr;
            if (warp == kTtSoftmaxWarps) {
              kr = reinterpret_cast<const float2*>(st + Codes::kOffKr)[lane];
              vr = reinterpret_cast<const float2*>(st + Codes::kOffVr)[lane];
            }
            __syncwarp();
            if (lane == 0) ts_arrive(&ring_free[rr.i]);
            rr.next();
            ok = is_v ? ts_wait(&v_free[rv.i], rv.phase ^ 1u, &s_bad) : ts_wait(&k_free[rk.i], rk.phase ^ 1u, &s_bad);
            if (!(ok = __all_sync(kFull, ok))) break;
            if (warp == kTtSoftmaxWarps) {  // the first of these warps: the row scales
              float* un = units_kv + slot * C::kUnitFloats;
              reinterpret_cast<float2*>(un)[lane] = make_float2(kr.x * p.scale_log2, kr.y * p.scale_log2);
              reinterpret_cast<float2*>(un + kTtKeys)[lane] = vr;
            }
            slot = slot + 1 == kTtUnitSlots ? 0 : slot + 1;
            uint8_t* out = smem + (is_v ? C::kOffV + rv.i * C::kOperand : C::kOffK + rk.i * C::kOperand);
            auto prepare = [&](auto clean_tag) {
              constexpr bool CLEAN = decltype(clean_tag)::value;
#pragma unroll
              for (int x = 0; x < kRounds; ++x) {
                const int r = r0 + x * kStep;
                const uint32_t word[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
                [[maybe_unused]] uint32_t b0 = 0, b1 = 0;
                if constexpr (FMT == kKvFmtNvfp4) {
                  const uint32_t both = e4m3x2_to_f16x2(scales[x]);
                  b0 = __byte_perm(both, both, 0x1010);
                  b1 = __byte_perm(both, both, 0x3232);
                }
#pragma unroll
                for (int y = 0; y < kChunks; ++y) {
                  uint32_t h[4];
                  if constexpr (FMT == kKvFmtNvfp4) {
                    e2m1x8_to_f16x2x4(word[y], h);
#pragma unroll
                    for (int z = 0; z < 4; ++z) h[z] = ts_hmul2(h[z], y < 2 ? b0 : b1);
                  } else {
                    ts_e4m3x4(word[2 * y], h[0], h[1]);
                    ts_e4m3x4(word[2 * y + 1], h[2], h[3]);
                  }
                  if constexpr (CLEAN) {
                    uint32_t bad = 0;
#pragma unroll
                    for (int z = 0; z < 4; ++z) h[z] = r < live ? ts_finite<FMT>(h[z], bad) : 0u;
                    if (bad) s_wild = 1u;
                  }
                  *reinterpret_cast<uint4*>(out + dst0[y] + x * kStep * 128) = make_uint4(h[0], h[1], h[2], h[3]);
                }
              }
            };
            if (busy && is_v && edge) prepare(std::true_type{});
            else if (busy) prepare(std::false_type{});
            tt_fence_async();
            __syncwarp();
            if (lane == 0) ts_arrive(is_v ? &v_full[rv.i] : &k_full[rk.i]);
            rk.next();
            rv.next();
          } else if (is_v) {
            ok = ts_wait(&v_raw[rv.i], rv.phase, &s_bad);
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
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTtSoftmaxRegs));
    const int quarter = (warp & 3) - (upper && warp >= 4 ? 2 : 0);
    TsWalk w;
    bool more = begin(w) && quarter >= 0 && quarter < active;
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;  // stream, row of its tile
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t s_count = 0, o_count = 0, end_phase = 0, o_end_phase = 0;  // scores seen, P tiles given, segments ended
    bool first_segment = true;
    int slot0 = 0;  // unit slot of the segment's first tile
    [[maybe_unused]] int tile0 = 0;  // the CTA's tiles before the segment
    bool ok = true;
    // Row of Q and of the context of row n of a pass of unit u.
    auto q_row = [&](int64_t b, int u, int n) {
      const int at = u % p.passes * p.rows_per_pass + n;
      return (b * p.tokens + at / p.group) * p.q_heads + static_cast<int64_t>(u / p.passes) * p.group + at % p.group;
    };
    for (; more && ok; more = w.next()) {
      const int b = w.b, kvh = w.u / p.passes, pass = w.u % p.passes, tiles = w.t1 - w.t0;
      const int past = PAGED ? ts_lengths(p, prefix)[b].x : ts_past(p, b);
      const int vis = PAGED ? ts_lengths(p, prefix)[b].y : ts_visible(p, b);
      const int n_first = pass * p.rows_per_pass, rows = min(p.rows_per_pass, nq - n_first);
      const bool shifted = upper;
      const int half = (rows + 1) / 2;
      // This thread's query row of the pass (out of [0, rows): none).
      const int n = SPLIT ? (r < half ? s * half + r : rows) : (shifted && s == 1 ? r - 64 : r);
      const bool has = n >= 0 && n < rows;
      const bool warp_has = __any_sync(kFull, has);
      const int tok = has ? (n_first + n) / p.group : 0;
      const int64_t q_row_own = q_row(b, w.u, n);
      if (!SPLIT && !first_segment) {  // both streams have read what the join left in the place of Q
        ok = ts_wait(&join_read, end_phase ^ 1u, &s_bad);
        if (!(ok = __all_sync(kFull, ok))) break;
      }
      first_segment = false;
      // ---- Q: this thread's row (SPLIT: all of it; else the panel of its stream)
      float own = kQuant ? 1.0f : p.scale_log2;
      // Eight lanes a row and panel, all loads in flight: a segment waits for these rows, and with a row per lane every
      // load touched 32 lines (48 tokens after 32 positions, BF16: 42.4 us so, 40.8 us as here).
      if (warp_has) {
        constexpr bool kHalves = !SPLIT && C::kPanels == 2;
        constexpr int kMine = SPLIT ? C::kPanels : 1;  // panels this stream stores
        const int64_t own_row = has ? q_row(b, w.u, n) : 0;
        const int held = __popc(__ballot_sync(kFull, has));
        const int first = kHalves ? s : 0;
        uint4 v[kMine][8], other[8];  // rows 4 i + lane / 8
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool there = 4 * i + (lane >> 3) < held;
          const uint4* src = reinterpret_cast<const uint4*>(p.q + __shfl_sync(kFull, own_row, 4 * i + (lane >> 3)) * D);
#pragma unroll
          for (int pn = 0; pn < kMine; ++pn)
            v[pn][i] = there ? __ldg(src + 8 * (first + pn) + (lane & 7)) : make_uint4(0u, 0u, 0u, 0u);
          if constexpr (kQuant && kHalves)
            other[i] = there ? __ldg(src + 8 * (1 - first) + (lane & 7)) : make_uint4(0u, 0u, 0u, 0u);
        }
        const int at0 = SPLIT ? s * kTtRows + (warp & 3) * 32 : (shifted ? 64 : 0) + __shfl_sync(kFull, n, 0);
        uint8_t* dst = smem + C::kOffQ + first * C::kQPanel;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 4 * i + (lane >> 3);
          [[maybe_unused]] float up = 1.0f;
          if constexpr (kQuant) {  // by a power of two, the row's largest element below 2^15
            uint32_t top = 0;
            auto largest = [&](const uint4& x) {
              top = __vmaxu2(top, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                           __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
            };
#pragma unroll
            for (int pn = 0; pn < kMine; ++pn) largest(v[pn][i]);
            if constexpr (kHalves) largest(other[i]);
            top = max(top & 0xffffu, top >> 16);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
            const int ex = static_cast<int>(top >> 7);
            const int e = (ex == 0 || ex == 255) ? 0 : min(14 - (ex - 127), 100);
            up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            const int mine = __shfl_sync(kFull, e, (lane & 3) * 8);  // row 4 i + lane % 4
            if ((lane >> 2) == i) own = __uint_as_float(static_cast<uint32_t>(127 - mine) << 23);
          }
          if (row < held && (SPLIT || kHalves || s == 0)) {
#pragma unroll
            for (int pn = 0; pn < kMine; ++pn) {
              uint4 x = v[pn][i];
              if constexpr (kQuant) {
                uint32_t* e = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  e[y] = ts_pack_f16(__uint_as_float(e[y] << 16) * up, __uint_as_float(e[y] & 0xffff0000u) * up);
              }
              *reinterpret_cast<uint4*>(dst + pn * C::kQPanel + tt_chunk(at0 + row, lane & 7)) = x;
            }
          }
        }
      }
      tt_fence_async();
      __syncwarp();
      if (lane == 0) ts_arrive(&q_full);

      float m = -INFINITY, l = 0.0f;  // the reference of the weights 2^(s - m), and their sum
      const uint8_t* mask_row = p.mask ? p.mask + b * p.mask_stride + static_cast<int64_t>(tok) * p.tokens : nullptr;
      int done = 0;  // jobs of this stream in the segment
      for (int i = SPLIT ? 0 : s; i < tiles && ok; i += SPLIT ? 1 : 2, ++done) {
        const int buf = s_count & 1;
        const int key0 = (w.t0 + i) * kTtKeys;
        // Keys of the tile this row sees, one bit each.  With a mask, a lane per key and a vote per token: a byte at a
        // time per row, it took a fifth of a one-tile segment's time.
        bool edge = key0 + kTtKeys > past;
        unsigned long long seen = ~0ull;
        if (edge) {
          if (!p.mask) {
            const int see = min(past + tok + 1, vis) - key0;
            seen = see <= 0 ? 0ull : see >= 64 ? ~0ull : (1ull << see) - 1;
          } else {
            // Opaque: what follows is worked out here, not kept in registers over the other tiles.
            int mine = tok;
            asm volatile("" : "+r"(mine));
            const uint8_t* mask_b = p.mask + b * p.mask_stride;
            auto sees = [&](int t, int pos) {
              if (pos < past) return true;
              return pos < vis && mask_b[static_cast<int64_t>(t) * p.tokens + (pos - past)] != 0;
            };
            // Tokens of the warp's rows (those that hold one come first).
            const int tok_lo = __shfl_sync(kFull, mine, 0), tok_hi = __reduce_max_sync(kFull, mine);
#pragma unroll 4
            for (int t = tok_lo; t <= tok_hi; ++t) {
              const uint32_t lo = __ballot_sync(kFull, sees(t, key0 + lane));
              const uint32_t hi = __ballot_sync(kFull, sees(t, key0 + 32 + lane));
              if (t == tok) seen = lo | static_cast<unsigned long long>(hi) << 32;
            }
          }
        }
        ok = ts_wait(&s_full[s][buf], (s_count >> 1) & 1, &s_bad);
        if (!(ok = __all_sync(kFull, ok))) break;
        tt_fence_after();
        if constexpr (PAGED) {
          const unsigned gone = s_gone[(tile0 + i) & (kTtGoneSlots - 1)];
          if (gone) {
            edge = true;
#pragma unroll
            for (int z = 0; z < kTtKeys / 16; ++z)
              if (gone >> z & 1u) seen &= ~(0xffffull << (16 * z));
          }
        }
        ++s_count;
        const uint32_t s_at = s_col(s, buf) + lanes;
        const float* unit = units_kv + ((slot0 + i) & (kTtUnitSlots - 1)) * C::kUnitFloats;
        auto tile = [&](auto edge_tag) {
          constexpr bool EDGE = decltype(edge_tag)::value;
          // 32 scores in units of own; unseen keys -inf.
          auto scores = [&](int h, float (&x)[32]) {
            tt_ld32(s_at + 32 * h, x);
            if constexpr (kQuant) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 u = *reinterpret_cast<const float4*>(unit + 32 * h + e);
                const float2 a = tt_mul2(make_float2(x[e], x[e + 1]), make_float2(u.x, u.y));
                const float2 c = tt_mul2(make_float2(x[e + 2], x[e + 3]), make_float2(u.z, u.w));
                x[e] = a.x;
                x[e + 1] = a.y;
                x[e + 2] = c.x;
                x[e + 3] = c.y;
              }
            }
            if constexpr (EDGE) {
              const uint32_t bits = static_cast<uint32_t>(seen >> (32 * h));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((bits >> e) & 1)) x[e] = -INFINITY;
            }
          };
          // 32 keys' P against m_ref into out (BF16: second terms into out2), the weights' sum into l_tile, over codes
          // the largest P into p_top.
          float l_tile = 0.0f;
          [[maybe_unused]] uint32_t p_top[2] = {0u, 0u};
          auto weights = [&](int h, const float (&x)[32], float m_ref, uint32_t (&out)[16],
                             [[maybe_unused]] uint32_t (&out2)[16]) {
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              [[maybe_unused]] float4 u;
              if constexpr (kQuant) u = *reinterpret_cast<const float4*>(unit + kTtKeys + 32 * h + e);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float2 y = tt_fma2(make_float2(x[e + 2 * i], x[e + 2 * i + 1]), make_float2(own, own),
                                   make_float2(-m_ref, -m_ref));
                y.x = ts_exp2(y.x);
                y.y = ts_exp2(y.y);
                sum[i] = tt_add2(sum[i], y);
                const int at = e / 2 + i;
                if constexpr (kQuant) {
                  y = tt_mul2(y, i ? make_float2(u.z, u.w) : make_float2(u.x, u.y));
                  if constexpr (EDGE) {  // a row that is not seen may have any scale
                    if (!((seen >> (32 * h + e + 2 * i)) & 1)) y.x = 0.0f;
                    if (!((seen >> (32 * h + e + 2 * i)) & 2)) y.y = 0.0f;
                  }
                  out[at] = ts_pack_f16(y.x, y.y);
                  p_top[i] = ts_largest(p_top[i], out[at]);
                } else {
                  out[at] = ts_pack_bf16(y.x, y.y);
                  out2[at] = ts_pack_bf16(y.x - __uint_as_float(out[at] << 16),
                                          y.y - __uint_as_float(out[at] & 0xffff0000u));
                }
              }
            }
            l_tile += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          };
          auto maxima = [&](const float (&x)[32], float (&mx)[4]) {
#pragma unroll
            for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], x[e]);
          };
          // First against the reference as it is; again, after it has moved, if that was too low.  (Leaving the first
          // pass out in a segment's first tile, where it is always too low, cost 160 to 270 bytes of spilled registers
          // and 16 tokens over NVFP4 154 -> 160 us.)
          float f = 1.0f;  // what the accumulator is to be scaled by
          bool over = false, again = false;  // over: this row's reference has to move
          if (warp_has) {
            uint32_t out[2][16];
            [[maybe_unused]] uint32_t out2[2][16];
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            const float m_ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[32];
              scores(h, x);
              if constexpr (!kQuant) maxima(x, mx);
              weights(h, x, m_ref, out[h], out2[h]);
            }
            if constexpr (kQuant) {
              const uint32_t p_max = ts_largest(p_top[0], p_top[1]) & 0x7fff7fffu;
              over = max(p_max & 0xffffu, p_max >> 16) >= kTsPLimit || l + l_tile > kTtSumLimit ||
                     (m == -INFINITY && (!EDGE || seen != 0ull));
            }
            [[maybe_unused]] float top = 0.0f;
            if constexpr (!kQuant) {
              top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * own;
              over = top > m + kTsSlack<FMT>;
            }
            over = over && has;
            again = __any_sync(kFull, over);
            if (again) {
              float next = top;
              if constexpr (kQuant) {  // by the largest score and the largest contribution of the tile
                float con = -INFINITY;
                top = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                  float x[16];
                  tt_ld16(s_at + 16 * h, x);
                  const float* u = unit + 16 * h;
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    x[e] *= u[e];
                    if (EDGE && !((seen >> (16 * h + e)) & 1)) x[e] = -INFINITY;
                    x[e] *= own;
                    top = fmaxf(top, x[e]);
                    con = fmaxf(con, x[e] + tt_log2(u[kTtKeys + e]));
                  }
                }
                // whole numbers: what was summed is rescaled without a rounding
                next = fmaxf(m, ceilf(fmaxf(con - kTtTop, top - kTtHead)));
                if (l + l_tile > kTtSumLimit) next = fmaxf(next, m + kTtSumStep);
              }
              if ((kQuant ? has : over) && top > -INFINITY) {  // over codes all rows: their next moves come later then
                f = m == -INFINITY ? 0.0f : ts_exp2(m - next);
                l *= f;
                m = next;
              }
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                tt_st16(s_at + tt_p_col<FMT>(2 * h), out[h]);
                if constexpr (!kQuant) tt_st16(s_at + tt_p_col<FMT>(2 * h) + 16, out2[h]);
              }
            }
          }
          if (again) {  // uniform in the warp
            // ---- the accumulator, once P V of the tile before is done
            if (done > 0 && __any_sync(kFull, f != 1.0f)) {
              // The scores of this job were issued after the P V of the job before last: one phase is in question.
              ok = ts_wait(&o_done[s], (o_count - 1) & 1, &s_bad);
              if (!(ok = __all_sync(kFull, ok))) return;
              tt_fence_after();
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                float o[16];
                tt_ld16(o_col(s) + lanes + c, o);
                uint32_t y[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(o[e] * f);
                tt_st16(o_col(s) + lanes + c, y);
              }
            }
            const float m_ref = m == -INFINITY ? 0.0f : m;
            l_tile = 0.0f;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              float x[32];
              scores(h, x);
              uint32_t out[16];
              [[maybe_unused]] uint32_t out2[16];
              weights(h, x, m_ref, out, out2);
              tt_st16(s_at + tt_p_col<FMT>(2 * h), out);
              if constexpr (!kQuant) tt_st16(s_at + tt_p_col<FMT>(2 * h) + 16, out2);
            }
          }
          l += l_tile;
          tt_wait_st();
          tt_fence_before();
          __syncwarp();
          if (lane == 0) ts_arrive(&p_full[s][buf]);
          ++o_count;
        };
        if (edge) tile(std::true_type{});
        else tile(std::false_type{});
      }
      slot0 = (slot0 + tiles) & (kTtUnitSlots - 1);
      if constexpr (PAGED) tile0 += tiles;
      // Every P V of the segment.  (Waiting on o_done here could miss it: it may be one or two phases on.)
      ok = ok && ts_wait(&o_end[s], o_end_phase, &s_bad);
      ok = __all_sync(kFull, ok);
      o_end_phase ^= 1u;
      tt_fence_after();
      // ---- the segment's (m, l, o)
      // Over codes, with l brought into [1, 2): the weights' own range may be far from 1.
      float unit_o = 1.0f;
      if constexpr (kQuant) {
        const int e = static_cast<int>(__float_as_uint(l) >> 23);
        if (e > 0 && e < 254) {
          unit_o = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e)
          l *= unit_o;
          m += static_cast<float>(e - 127);
        }
      }
      float4* area = reinterpret_cast<float4*>(smem + C::kOffQ);  // [D / 4][64 rows]
      if (!SPLIT) {
        // Every MMA of the segment has read its Q.  Where the streams' rows lie in different lanes, stream 0
        // joins the first half of the columns and stream 1 the second, each reading the other's accumulator in the
        // place of Q (16 tokens over 32,000 positions, NVFP4: 165 us with stream 0 alone, 160 us so).  Else stream 0
        // joins all, reading both in tensor memory (32 tokens, E4M3: halves took 66 us, this 64).
        __syncwarp();
        if (lane == 0) ts_arrive(&seg_done);
        ok = ok && ts_wait(&seg_done, end_phase, &s_bad);
        ok = __all_sync(kFull, ok);
        if (ok && warp_has) {
          if (done > 0 && shifted) {
#pragma unroll 1
            for (int c = (1 - s) * (D / 2), i = 0; i < D / 2; c += 16, i += 16) {
              float o[16];
              tt_ld16(o_col(s) + lanes + c, o);
              if (has)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  area[(c / 4 + e) * 64 + n] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
          if (has) join[s][n] = make_float4(m, l, unit_o, 0.0f);
        }
        tt_fence_before();
        __syncwarp();
        if (lane == 0) ts_arrive(&join_ready);
        ok = ok && ts_wait(&join_ready, end_phase, &s_bad);
        ok = __all_sync(kFull, ok);
        tt_fence_after();
        end_phase ^= 1u;
      }
      if (ok && warp_has) {
        float f_own = unit_o, f_other = 0.0f, mj = m, lj = l;
        const bool two = !SPLIT && tiles > 1;  // stream 1 had a tile
        if constexpr (!SPLIT) {
          const float4 none = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
          const float4 j0 = has ? join[0][n] : none, j1 = has && two ? join[1][n] : none;
          mj = fmaxf(j0.x, j1.x);
          const float a0 = j0.x == -INFINITY ? (j0.y == 0.0f ? 0.0f : 1.0f) : ts_exp2(j0.x - mj);
          const float a1 = j1.x == -INFINITY ? (j1.y == 0.0f ? 0.0f : 1.0f) : ts_exp2(j1.x - mj);
          lj = j0.y * a0 + j1.y * a1;
          f_own = s == 0 ? j0.z * a0 : j1.z * a1;
          f_other = s == 0 ? j1.z * a1 : j0.z * a0;
        }
        const bool whole = w.t0 == 0 && w.t1 == w.nt;
        int n_tiles, G, x0;
        range(n_tiles, G, x0);
        const int64_t slot = 2 * static_cast<int64_t>(cta) + (w.x == x0 ? 0 : 1);
        if (!whole && tid == 0) ts_write_slot<PAGED>(p, n_tiles, G, cta, x0, w);
        const bool padding = PAGED && tok >= ts_tokens<PAGED>(p, b);
        if (padding) lj = f_own = f_other = 0.0f;
        const float inv = lj == 0.0f ? 0.0f : __fdiv_rn(1.0f, lj);
        const int64_t v_row = (b * p.kv_heads + kvh) * p.capacity;
        // Infinities and NaN of V that were taken out, for the rows that see them: 16 columns.  They were taken out of
        // whole tiles, so the first such tile's committed rows, before P_b, count too.
        auto add_wild = [&](int c, float (&o)[16]) {
          const int first = max(past / kTtKeys * kTtKeys, w.t0 * kTtKeys), last = min(vis, w.t1 * kTtKeys);
          for (int pos = first; pos < last; ++pos) {
            if (!tree_sees(mask_row, tok, pos - past)) continue;
            int64_t row = v_row + pos;
            if constexpr (PAGED) {
              const int page = paged_page(p.pg, b, pos);
              if (page < 0) continue;
              row = (static_cast<int64_t>(page) * p.kv_heads + kvh) * p.pg.page_size + pos % p.pg.page_size;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x = tt_v_global<D, FMT>(p.v, row, c + e);
              if (!isfinite(x)) o[e] += x;
            }
          }
        };
        if constexpr (SPLIT) {
          // 32 columns at a time, turned in the place of this warp's own Q rows so that a store's lanes write whole
          // lines; with a row per lane a store touches 32 (48 tokens after 32 positions, BF16: 37.8 -> 36.2 us).
          // Without SPLIT the joins leave half of the warps at it, and the turn costs more than it saves
          // (16 tokens after 1,000 positions, NVFP4: 35.9 -> 41.2 us).
          uint8_t* turn = smem + C::kOffQ + warp * 4096;
          const int n0 = __shfl_sync(kFull, n, 0), held = __popc(__ballot_sync(kFull, has));
          const float f = whole ? f_own * inv : f_own;
          float* part = p.part_o + (slot * p.rows_per_pass + n0 + (lane >> 3)) * D + 4 * (lane & 7);
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
#pragma unroll 1
            for (int h = c; h < c + 32; h += 16) {
              float o[16];
              tt_ld16(o_col(s) + lanes + h, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = f == 0.0f ? 0.0f : o[e] * f;
              if (has && s_wild && f != 0.0f) add_wild(h, o);
              if (has)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  *reinterpret_cast<float4*>(turn + tt_chunk(lane, (h - c) / 4 + e)) =
                      make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            __syncwarp();
            if (whole) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int row = i * 8 + (lane >> 2), ch = (lane & 3) * 2;
                const int64_t to = __shfl_sync(kFull, q_row_own, row);
                if (row < held) {
                  const float4 x = *reinterpret_cast<const float4*>(turn + tt_chunk(row, ch));
                  const float4 y = *reinterpret_cast<const float4*>(turn + tt_chunk(row, ch + 1));
                  *reinterpret_cast<uint4*>(p.ctx + to * D + c + 4 * ch) =
                      make_uint4(ts_pack_bf16(x.x, x.y), ts_pack_bf16(x.z, x.w), ts_pack_bf16(y.x, y.y),
                                 ts_pack_bf16(y.z, y.w));
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int row = i * 4 + (lane >> 3);
                if (row < held)
                  *reinterpret_cast<float4*>(part + c + i * 4 * D) =
                      *reinterpret_cast<const float4*>(turn + tt_chunk(row, lane & 7));
              }
            }
            __syncwarp();
          }
        } else {
#pragma unroll 1
          for (int c = shifted ? s * (D / 2) : s * D, i = 0; i < (shifted ? D / 2 : D) && c < D; c += 16, i += 16) {
            float o[16], o1[16];
            if (s == 0 || two) {
              tt_ld16(o_col(s) + lanes + c, o);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = 0.0f;
            }
            if (s == 0 && !two) {
#pragma unroll
              for (int e = 0; e < 16; ++e) o1[e] = 0.0f;
            } else if (!shifted) {
              tt_ld16(o_col(1 - s) + lanes + c, o1);
            } else if (has) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 x = area[(c / 4 + e) * 64 + n];
                o1[4 * e] = x.x;
                o1[4 * e + 1] = x.y;
                o1[4 * e + 2] = x.z;
                o1[4 * e + 3] = x.w;
              }
            }
            if (!has) continue;  // the next tt_ld16 brings the lanes together again
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = (f_own == 0.0f ? 0.0f : o[e] * f_own) + (f_other == 0.0f ? 0.0f : o1[e] * f_other);
            if (s_wild && !padding) add_wild(c, o);
            if (whole) {
              uint4* dst = reinterpret_cast<uint4*>(p.ctx + q_row_own * D + c);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t x[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  x[y] = lj == 0.0f ? 0u : ts_pack_bf16(o[8 * e + 2 * y] * inv, o[8 * e + 2 * y + 1] * inv);
                dst[e] = make_uint4(x[0], x[1], x[2], x[3]);
              }
            } else {
              float4* dst = reinterpret_cast<float4*>(p.part_o + (slot * p.rows_per_pass + n) * D + c);
#pragma unroll
              for (int e = 0; e < 4; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
        }
        if (has && !whole && (SPLIT || s == 0)) p.part_ml[slot * p.rows_per_pass + n] = make_float2(mj, lj);
      }
      tt_fence_before();
      __syncwarp();
      if (!SPLIT && lane == 0) ts_arrive(&join_read);
    }
  }
  // Where a wait gave up, the MMAs in flight end before their tiles and tensor memory go to another.  (Here, not in the
  // issuing warps' branch: there it took 16 tokens over NVFP4 from 157 to 162 us.)
  if (__any_sync(kFull, s_bad) && (warp == kTtMmaWarp || warp == kTtMmaWarp + 2)) {
    if (tt_elect()) {  // the lane that issued them: the election is the same each time
      uint64_t* bar = &drained[(warp - kTtMmaWarp) / 2];
      tt_commit(bar);
      ts_landed(bar, 0);
    }
    __syncwarp();
  }
  tt_fence_before();
  __syncthreads();
  if (warp == kTtMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace nvfp4da
