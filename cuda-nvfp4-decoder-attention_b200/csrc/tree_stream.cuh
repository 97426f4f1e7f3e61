// Tree attention at HBM rate: a persistent, TMA-fed tensor-core kernel that
// reads a BF16, E4M3 or NVFP4 cache in its own format (head_dim 64, 128, 256).
// Semantics: tree_attention.cuh.
//
// Work decomposition.  The group * T query rows of one (sequence, KV head) are
// cut into passes of RP rows (nearly always one pass).  Every (sequence, KV
// head, pass) owns the tiles that its P_b + T keys fill, of 64 positions over
// BF16 and of 128 over codes; all of them are laid end to end and one CTA per SM
// takes an equal contiguous range of that line, so every SM streams the same
// bytes whatever the lengths.  A CTA's part of one unit either is the whole unit
// (the result is written) or leaves a partial (o, m, l): only a CTA's first and
// last parts can be partial, so it has two slots.  tree_stream_combine_kernel
// joins a unit's partials in CTA order.
//
// Per CTA: two warps fill a ring of stages, one with K and one with V tiles (TMA,
// 128-byte swizzle) and the scales of both (16-byte asynchronous copies by all of
// its lanes); two more join and write what the consumers leave of a segment.  NW
// consumer warps: RC row chunks of 8 NG query rows, NW / RC position warps per
// chunk; a warp takes 16-position slices, whole tiles alternating between groups
// of four position warps.  With x^T for a fragment that holds positions or head
// elements in its 16 rows and queries in its 8 columns:
//   S^T[pos, q] = K[pos, :] . Q^T      mma.m16n8k16, FP32 accumulators
//   O^T[d, q]  += V^T[d, pos] P^T
// The element k of an MMA step may be any element of the head as long as K and
// Q agree, and a row of O^T any element d: a lane of K takes D/4 consecutive
// elements of its row, a lane of V takes D/8 consecutive elements of its four
// positions, so codes are read 8 or 16 bytes at a time and decoded in
// registers; nothing is written back to shared memory.
//
// Numerics.  Codes (times the NVFP4 block scale) are exact in FP16; the query
// row is scaled to FP16 by the power of two that brings its largest element to
// [2^14, 2^15), 2^100 at most: its 8 bits are exact from 2^-31 of that element on,
// smaller ones are off by 2^-25 of the scaled row (2^-39 of it) at most; the row
// scale of K multiplies the FP32 score.  P goes to FP16 as
// p_j gamma_j / G 2^5, where G follows the largest contribution p_j gamma_j that
// the query has met (>= 2^-100): 11 significant bits down to 2^-19 of that
// contribution, absolute steps of 2^-29 of it below.  (With the largest gamma_j
// in the place of G, a key that carries nearly all of the weight lost its bits
// when its row of V was small beside one that weighs nothing.)  Over BF16 caches
// Q and V stay BF16 and P is split into two BF16 terms.  The softmax runs in base
// 2; its reference m moves only when a score passes it, to 2^10 above that score
// (BF16: when one passes it by 2^20, to the score), and G only when a contribution
// passes it by 2^10, so most slices need neither a reduction nor a rescale.  m, l,
// o and all sums are FP32; o is held in units of G, which shrinks with p_j when m
// moves, so that a move of m leaves o as it is.
//
// Slices that reach P_b (drafted tokens, the sequence's end) take a second
// instantiation that applies the mask, drops positions past the end and zeroes
// infinities and NaN in V before the MMA (0 * NaN would reach queries that do
// not see the row); queries that do see such an element get it added after.
//
// What bounds it: a single token over ragged E4M3 caches (64 sequences x 6 heads,
// 1,024 to 8,191 positions, 460 MB) takes 92 us, 5.0 TB/s, 0.76 of a copy; of
// that the launches, the first tiles' latency and the join of partials are some
// 12 us, the rest streams at 0.87.  Over NVFP4 (8 sequences, 32,768 positions)
// 71 us, 3.4 TB/s: decoding codes to FP16 in registers, 43 % of the issue slots
// and the latency between them with two warps a scheduler, no longer the bytes.
// G by the largest row scale alone, checked before the exponentials, took 70 us there.
// 12 or 16 consumer warps, for which registers suffice with one slice at a time,
// were no faster.
//
// PAGED (paged_kv.cuh): the cache is a pool of pages, position j of sequence b row
// j % S of page table[b, j / S].
//   tiles     come in boxes of 2^k positions (the largest that divides the page and
//             the tile), each a TMA copy of its own; with more than one a tile, two
//             warps copy K and two V, since a thread takes some 200 cycles to issue
//             a copy.  Copied 16 bytes a lane instead, E4M3 in pages of 16 took 176
//             us where the TMA unit took 111.  A warp looks 32 boxes up at once.
//   pages     that the table does not name, and padding (counts): the loading warp
//             marks a tile's 16-position slices that are not there, consumers leave
//             them out; a padding row's context is zeros.
//   the line  is cut by weight, a segment counting kTsSegment tiles beside its own:
//             64 E4M3 sequences of 10 to 2,000 positions, pages of 16, 59 us unweighted,
//             47 so.
//   a segment's start and end: lengths stand in shared memory, four warps join its
//             rows, and its last slices are taken one at a time, half of the code to
//             fetch (a segment had missed the instruction cache at every third
//             request).
// 64 sequences x 6 heads, 1,024 to 8,191 positions, one token: BF16 142 us, 6.3
// TB/s, 0.96 of a copy; E4M3 in pages of 16 94 us, 4.9 TB/s (no arithmetic at all:
// 10 us less); 8 x 32,768 of NVFP4 78 us: the ALU pipe's decoding (64 conversions
// and 36 unpackings a slice), 45 % of the issue slots.  Head dimension 256 (1,024 to
// 8,191 positions): BF16 290 us, 0.98 of a copy, E4M3 171, NVFP4 166; its instances
// spill 80 to 132 bytes a thread, that of three groups of E4M3 at 64 44 bytes.
//
// Waits are bounded: one that lasts a second records kErrBarrierTimeout in
// g_tree_errors, and every role of the CTA leaves (its results are then garbage;
// the GPU stays usable).  The loading warps leave only when what they copy into
// shared memory has landed, or after a further limit.
#pragma once

#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kv_quant.cuh"
#include "paged_kv.cuh"
#include "tree_attention.cuh"

namespace nvfp4da {

static __device__ unsigned g_tree_errors;  // of the translation unit's kernels

// Positions per stage: with 64, the 4 KB pieces of NVFP4 codes reached two
// thirds of the HBM rate even with nothing else to do.
template <int FMT>
constexpr int kTsTile = FMT == kKvFmtBf16 ? 64 : 128;
// PAGED: what a segment costs beside its tiles, in tiles.  us for 0, 2, 4, 6 of them, 24 query heads over 6 KV heads:
// 64 sequences of 10 to 2,000 positions, pages of 32, BF16 76, 63, 63, 64, E4M3 86, 55, 49, 49, NVFP4 89, 61, 57, 54 (as
// the kernel was when this was chosen; with the last slices taken one at a time 0 costs less, see above); of 1,024 to
// 8,191 E4M3 113, 109, 111, 114; 16 of 100 to 30,000 NVFP4 90, 80, 78, 78.
template <int FMT>
constexpr int kTsSegment = FMT == kKvFmtBf16 ? 3 : 4;
constexpr int kTsPagedRegs = 176, kTsPagedOtherRegs = 80;  // 256 * 176 + 256 * 80 = 512 * 128
constexpr int kTsMaxBatch = 1024;  // sequences whose prefix shared memory holds
// A score may pass the reference m by kTsSlack (log2), and m moves to kTsLift
// above the score that passed it.  Over codes p_j <= 1 then, so that p_j gamma_j
// cannot overflow; it may pass G until P in FP16, kTsPScale p_j gamma_j / G,
// reaches kTsPLimit.  BF16 terms have the range of FP32.
template <int FMT>
constexpr float kTsSlack = FMT == kKvFmtBf16 ? 20.0f : 0.0f;
template <int FMT>
constexpr float kTsLift = FMT == kKvFmtBf16 ? 0.0f : 10.0f;
constexpr float kTsPScale = 32.0f;
constexpr uint32_t kTsPLimit = 0x7800u;  // 2^15 in FP16
constexpr float kTsMinUnit = 7.88860905e-31f;  // 2^-100

template <int D, int FMT, int NG, int NW, int SL, int TILE = kTsTile<FMT>, bool PAGED = false>
struct TsCfg {
  static_assert(D == 64 || D == 128 || D == 256, "head_dim 64, 128 or 256");
  // Consumers, two loading and two joining warps; PAGED: four of each.
  static constexpr int kLoaders = PAGED ? 4 : 2, kJoiners = PAGED ? 4 : 2;
  static constexpr int kThreads = (NW + kLoaders + kJoiners) * 32;
  static constexpr int kRowBytes = FMT == kKvFmtBf16 ? 2 * D : (FMT == kKvFmtE4m3 ? D : D / 2);
  static constexpr uint32_t kCodes = TILE * kRowBytes;  // one of K, V
  static constexpr uint32_t kBlockScales = FMT == kKvFmtNvfp4 ? TILE * (D / 16) : 0;
  static constexpr uint32_t kRowScales = FMT == kKvFmtBf16 ? 0 : TILE * 4;
  static constexpr uint32_t kOffV = kCodes, kOffKb = 2 * kCodes, kOffVb = kOffKb + kBlockScales,
                            kOffKr = kOffVb + kBlockScales, kOffVr = kOffKr + kRowScales;
  static constexpr uint32_t kTx = kOffVr + kRowScales;  // bytes a stage receives
  static constexpr uint32_t kStage = (kTx + 1023) / 1024 * 1024;
  static constexpr int kRows = 8 * NG;                               // query rows per warp
  // What the consumer warps leave of a segment for the joining warps: o, m, l;
  // twice, so that they go on to the next segment, where it fits.
  static constexpr int kJoins = NG == 1 && D <= 128 ? 2 : 1;
  static constexpr int kJoinStride = D + (FMT == kKvFmtBf16 ? 8 : 2);  // floats between rows (bank conflicts)
  static constexpr uint32_t kJoinO = NW * kRows * kJoinStride * 4;
  static constexpr uint32_t kComb = kJoins * (kJoinO + 2 * NW * kRows * 4);
  static constexpr int kTurns = TILE / 16 / SL;                              // warps' turns per tile
  static constexpr int kGroups = NW / kTurns;                        // most tile groups
  // PAGED: a sequence's P_b and end beside its prefix.
  static constexpr uint32_t kPerSequence = PAGED ? 12 : 4;
  static constexpr int kFit = static_cast<int>(((PAGED ? 209u : 217u) * 1024 - kComb) / kStage);
  // A whole number of groups: the CTA's n-th tile goes to stage n % kStages and
  // group n % groups, so every stage serves one group only.
  static constexpr int kStages = (kFit > 14 ? 14 : kFit) / kGroups * kGroups;
  static_assert(kStages >= 2, "two stages at least");
  static constexpr uint32_t kOffComb = kStages * kStage;
  static constexpr uint32_t kOffBar = kOffComb + kComb;
  static constexpr uint32_t kOffPrefix = kOffBar + (2 * kStages + 2 * kJoins) * 8;
  static constexpr uint32_t bytes(int batch) { return kOffPrefix + kPerSequence * (batch + 1) + 1024; }
};

struct TreeStreamParams {
  const uint16_t* q;
  KvStore k, v;  // scales; the codes come through the tensor maps
  const uint8_t* mask;
  int64_t mask_stride;
  uint16_t* ctx;
  int batch, tokens, q_heads, kv_heads, group;
  int64_t capacity;
  int64_t past_length;
  const int64_t* past_lengths;
  float scale_log2;    // log2(e) / sqrt(D)
  int row_chunks;      // RC: power of two, <= NW
  int rows_per_pass;   // RP = 8 NG RC
  int passes;
  int grid;            // CTAs of the streaming kernel
  float* part_o;       // [2 grid][RP][D]: slots 2 CTA (its first segment) and 2 CTA + 1 (its last)
  float2* part_ml;     // [2 grid][RP]
  int4* part_slots;    // [2 grid]: see ts_write_slot
  PagedView pg;        // PAGED: the block table; the stores are a pool's, capacity = M * S
  int seg;             // PAGED: kTsSegment
  int loaders;         // PAGED: warps that copy K and V, 2 or 4 (a tile then has two boxes at least)
  int box_log2;        // PAGED: positions that one copy brings, a power of two >= 16 that divides the page and the tile
};

// ---------------------------------------------------------------- PTX
__device__ __forceinline__ void ts_tma_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}
// 16 bytes by this thread, and its arrival on `bar` once all it copied so is there.
__device__ __forceinline__ void ts_copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// The same, zeros where there is nothing to copy (`src` is valid all the same).
__device__ __forceinline__ void ts_copy16_or_zeros(void* dst, const void* src, bool copy) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(copy ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void ts_copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ts_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint32_t ts_transpose(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float ts_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int FMT>
__device__ __forceinline__ void ts_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if constexpr (FMT == kKvFmtBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ts_ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ts_ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t ts_pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t ts_pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t ts_hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Of each FP16 half, the one of larger magnitude (with some sign); NaN only where both are.
__device__ __forceinline__ uint32_t ts_largest(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two packed pairs of E4M3 -> two f16x2.
__device__ __forceinline__ void ts_e4m3x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}

// ---------------------------------------------------------------- bounded waits
// Nanoseconds, modulo 2^32: for differences of a few seconds at most.
__device__ __forceinline__ uint32_t ts_now() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}
// Gives up when another role has (`bad`) or after one second.
__device__ __forceinline__ bool ts_wait(uint64_t* bar, uint32_t parity, volatile unsigned* bad) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = ts_now();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 0) {
      if (*bad) return false;
      if (ts_now() - t0 > 1000000000u) {
        atomicOr(&g_tree_errors, static_cast<unsigned>(kErrBarrierTimeout));
        *bad = 1u;
        return false;
      }
    }
  }
}
// The last of n fills, in turn, of N buffers that went to buffer i, and the parity of its phase.
__host__ __device__ constexpr int ts_last_fill(int n, int N, int i) { return n - 1 - (n - 1 - i) % N; }
__host__ __device__ constexpr uint32_t ts_fill_parity(int fill, int N) { return static_cast<uint32_t>(fill / N) & 1u; }
static_assert(ts_last_fill(3, 4, 0) == 0 && ts_last_fill(3, 4, 2) == 2 && ts_last_fill(4, 4, 3) == 3 &&
                  ts_last_fill(6, 4, 1) == 5 && ts_last_fill(6, 4, 2) == 2 && ts_last_fill(9, 4, 0) == 8 &&
                  ts_fill_parity(3, 4) == 0 && ts_fill_parity(4, 4) == 1 && ts_fill_parity(8, 4) == 0,
              "fills of a ring");
// Waits for the phase, whoever has given up, but 20 ms at most.
__device__ __forceinline__ void ts_landed(uint64_t* bar, uint32_t parity) {
  const uint32_t t0 = ts_now();
  while (!mbar_try_wait(bar, parity) && ts_now() - t0 < 20000000u) {
  }
}
// Of n fills of a ring of N buffers, the last of each.
template <int N>
__device__ __forceinline__ void ts_all_landed(uint64_t* bars, int n) {
  for (int i = 0; i < N && i < n; ++i) ts_landed(&bars[i], ts_fill_parity(ts_last_fill(n, N, i), N));
}
// This thread's copies by ts_copy16.
__device__ __forceinline__ void ts_copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Byte offset o of a tile of 128-byte lines, 16-byte chunks swizzled by line.
__device__ __forceinline__ uint32_t ts_swz(uint32_t o) { return o ^ ((o >> 3) & 0x70u); }

// The 16-bit halves of w whose exponent is all ones (FP16 or BF16) become 0;
// `bad` collects them (bit 0: low half, bit 1: high half).
template <int FMT>
__device__ __forceinline__ uint32_t ts_finite(uint32_t w, uint32_t& bad) {
  constexpr uint32_t e = FMT == kKvFmtBf16 ? 0x7f80u : 0x7c00u;
  if ((w & e) == e) {
    bad |= 1u;
    w &= 0xffff0000u;
  }
  if (((w >> 16) & e) == e) {
    bad |= 2u;
    w &= 0x0000ffffu;
  }
  return w;
}

// ---------------------------------------------------------------- the walk over one CTA's range
struct TsWalk {
  const int* prefix;  // [B + 1]: tiles before sequence b (all its units)
  int units;          // per sequence
  int x, x_end;
  int b, u;
  int t0, t1, nt;  // this segment's tiles [t0, t1) of nt in the unit
  __device__ bool begin(const int* pre, int batch, int per_seq, int x0, int x1) {
    prefix = pre;
    units = per_seq;
    x = x0;
    x_end = x1;
    if (x >= x_end) return false;
    int lo = 0, hi = batch - 1;  // the last b with prefix[b] <= x (every sequence has a tile)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    nt = (prefix[b + 1] - prefix[b]) / units;
    const int within = x - prefix[b];
    u = within / nt;
    t0 = within % nt;
    t1 = min(nt, t0 + (x_end - x));
    return true;
  }
  __device__ bool next() {
    x += t1 - t0;
    if (x >= x_end) return false;
    if (++u == units) {
      u = 0;
      ++b;
      nt = (prefix[b + 1] - prefix[b]) / units;
    }
    t0 = 0;
    t1 = min(nt, x_end - x);
    return true;
  }
};

// P_b and the positions of sequence b that any of its drafted tokens may see
// (both fit 32 bits: a cache has fewer than 2^31 rows).
__device__ __forceinline__ int ts_past(const TreeStreamParams& p, int b) {
  return static_cast<int>(tree_past(p.past_lengths, p.past_length, b, p.capacity));
}
// Tokens of sequence b that are no padding.
template <bool PAGED>
__device__ __forceinline__ int ts_tokens(const TreeStreamParams& p, int b) {
  if constexpr (PAGED) return paged_count(p.pg, b, p.tokens);
  return p.tokens;
}
template <bool PAGED = false>
__device__ __forceinline__ int ts_visible(const TreeStreamParams& p, int b) {
  const int tokens = ts_tokens<PAGED>(p, b);
  if (PAGED && tokens == 0) return 0;
  return static_cast<int>(min(static_cast<int64_t>(ts_past(p, b)) + tokens, p.capacity));
}

// First tile of CTA c of g over n tiles.
__device__ __forceinline__ int ts_first_tile(int n, int c, int g) {
  return static_cast<int>(static_cast<long long>(n) * c / g);
}

// PAGED: P_b and the end of every sequence, behind the prefix in shared memory (read from global memory, they were
// a latency at the start of every segment).
__device__ __forceinline__ int2* ts_lengths(const TreeStreamParams& p, int* prefix) {
  return reinterpret_cast<int2*>(prefix + (p.batch + 2) / 2 * 2);
}

// The tiles before every sequence, into prefix[0 .. B]; all threads of the block.
template <bool PAGED = false>
__device__ __forceinline__ void ts_prefix(const TreeStreamParams& p, int units, int tile, int* prefix) {
  for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
    const int vis = ts_visible<PAGED>(p, b);
    int tiles = (vis + tile - 1) / tile;
    if constexpr (PAGED) {
      tiles = max(tiles, 1);  // a sequence of nothing but padding: one that nobody sees
      ts_lengths(p, prefix)[b] = make_int2(ts_past(p, b), vis);
    }
    prefix[b + 1] = tiles * units;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int carry = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int b = base + lane;
      int v = b < p.batch ? prefix[b + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFull, v, o);
        if (lane >= o) v += u;
      }
      if (b < p.batch) prefix[b + 1] = carry + v;
      carry += __shfl_sync(kFull, v, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
}

// PAGED: the line is cut by weight instead, a segment counting as kTsSegment tiles
// beside its own, so that a CTA with many short units is not the last to end.
// On the weighted line a unit takes kTsSegment places and then one a tile; tile t
// belongs to the CTA that holds its place.
__device__ __forceinline__ int ts_places(const TreeStreamParams& p, const int* prefix, int units) {
  return prefix[p.batch] + p.seg * units * p.batch;
}
// First tile (on the line of tiles) of CTA c of g.
__device__ __forceinline__ int ts_first_tile_weighted(const TreeStreamParams& p, const int* prefix, int units, int c,
                                                      int g) {
  const int x = ts_first_tile(ts_places(p, prefix, units), c, g);
  if (c == g) return prefix[p.batch];
  int lo = 0, hi = p.batch - 1;  // the last sequence that begins at or before x
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] + p.seg * units * mid <= x) lo = mid;
    else hi = mid - 1;
  }
  const int nt = (prefix[lo + 1] - prefix[lo]) / units, within = x - prefix[lo] - p.seg * units * lo;
  const int u = within / (nt + p.seg), o = within % (nt + p.seg);
  return prefix[lo] + u * nt + max(0, o - p.seg);
}

// CTA (of g over n tiles, CTA c owning [c n / g, (c + 1) n / g)) that holds tile x.
__device__ __forceinline__ int ts_cta_of(int x, int n, int g) {
  return static_cast<int>(((static_cast<long long>(x) + 1) * g - 1) / n);
}

// What a slot of partials holds: the unit and its CTAs, where the slot is the
// first part of a unit that several CTAs share; unit -1 otherwise.
template <bool PAGED = false>
__device__ __forceinline__ void ts_write_slot(const TreeStreamParams& p, int n_tiles, int G, int cta, int x0,
                                              const TsWalk& w) {
  const bool first = w.x == x0;
  const bool starts = w.t0 == 0 && w.t1 < w.nt;  // the unit's first part, more to come
  int end = w.x - w.t0 + w.nt - 1;               // the unit's last tile
  if constexpr (PAGED) end += p.seg * (w.units * w.b + w.u + 1);  // its place; n_tiles: places
  const int last = ts_cta_of(end, n_tiles, G);
  p.part_slots[2 * cta + (first ? 0 : 1)] =
      starts ? make_int4(w.b, w.u, cta, last) : make_int4(-1, 0, 0, 0);
}

// Element d of position r (in the tile) of V as the MMA saw it, before ts_finite.
template <int D, int FMT>
__device__ __forceinline__ float ts_v_element(const uint8_t* vt, const uint8_t* vb, int r, int d) {
  if (FMT == kKvFmtBf16) {
    const uint32_t o = (d >> 6) * (kTsTile<FMT> * 128) + ts_swz(r * 128 + (d & 63) * 2);
    return bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(vt + o));
  }
  if (FMT == kKvFmtE4m3) return f16x2_to_f32x2(e4m3x2_to_f16x2(vt[ts_swz(r * D + d)])).x;
  const uint32_t byte = vt[ts_swz(r * (D / 2) + d / 2)];
  const float2 pair = f16x2_to_f32x2(e2m1x2_to_f16x2(byte));
  return ((d & 1) ? pair.y : pair.x) * f16x2_to_f32x2(e4m3x2_to_f16x2(vb[r * (D / 16) + d / 16])).x;
}

// The scales of the TILE rows from `row` on, by one warp; rows past the cache's
// last are left out (they belong to no position that is seen).
template <int D, int FMT, typename Cfg, int TILE>
__device__ __forceinline__ void ts_load_scales(uint8_t* st, const TreeStreamParams& p, int64_t row, int64_t rows,
                                               int lane) {
  const int left = static_cast<int>(min(rows - row, static_cast<int64_t>(TILE)));
  if constexpr (FMT == kKvFmtNvfp4) {
#pragma unroll
    for (uint32_t i = 0; i < Cfg::kBlockScales; i += 512) {
      const uint32_t o = i + lane * 16;
      if (o < static_cast<uint32_t>(left) * (D / 16)) {
        ts_copy16(st + Cfg::kOffKb + o, p.k.block_scales + row * (D / 16) + o);
        ts_copy16(st + Cfg::kOffVb + o, p.v.block_scales + row * (D / 16) + o);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TILE; i += 128) {
    const int r = i + lane * 4;
    if (r < left) {
      ts_copy16(st + Cfg::kOffKr + r * 4, p.k.row_scales + row + r);
      ts_copy16(st + Cfg::kOffVr + r * 4, p.v.row_scales + row + r);
    }
  }
}

// ---------------------------------------------------------------- tiles of a paged cache
// Where a tile's boxes (2^box_log2 positions each) stand.  A lane looks up one box:
// 32 / boxes tiles at a time, the next ones while these are fetched, so that the
// table's latency is not in the way of the copies.
template <int TILE>
struct TsBoxes {
  int box_log2, per_log2, tiles;  // of a box's positions, a tile's boxes; tiles that 32 lanes hold
  int cur, next, t0;   // this lane's box of tiles t0 .. and of those behind them: its first row of the pool, -1: none
  int b, kvh, vis, t_end;
  __device__ int look(const TreeStreamParams& p, int t, int lane) const {
    const int pos = t * TILE + (lane << box_log2), of = t + (lane >> per_log2);
    if (pos >= vis || of >= t_end) return -1;
    const int page = paged_page(p.pg, b, pos);
    return page < 0 ? -1 : (page * p.kv_heads + kvh) * p.pg.page_size + pos % p.pg.page_size;
  }
  __device__ void begin(const TreeStreamParams& p, int b_, int kvh_, int vis_, int t, int t1, int lane) {
    box_log2 = p.box_log2;
    per_log2 = (TILE == 64 ? 6 : 7) - box_log2;
    tiles = 32 >> per_log2;
    b = b_;
    kvh = kvh_;
    vis = vis_;
    t0 = t;
    t_end = t1;
    cur = look(p, t, lane);
    next = look(p, t + tiles, lane);
  }
  // For tile t, in order; all lanes.
  __device__ void advance(const TreeStreamParams& p, int t, int lane) {
    if (t < t0 + tiles) return;
    t0 += tiles;
    cur = next;
    next = look(p, t0 + tiles, lane);
  }
  // The first row of position r's box (r modulo the tile); all lanes.
  __device__ int row(int t, int r) const { return __shfl_sync(kFull, cur, ((t - t0) << per_log2) + ((r & (TILE - 1)) >> box_log2)); }
};

// ts_load_scales of K or of V (`from`, to `blocks` and `rows`) for a tile whose boxes stand apart; zeros where there is
// none.
template <int D, int FMT, typename Cfg, int TILE>
__device__ __forceinline__ void ts_load_scales_paged(uint8_t* blocks, uint8_t* rows, const KvStore& from,
                                                     const TsBoxes<TILE>& at, int t, int lane) {
  const int in_box = (1 << at.box_log2) - 1;
  if constexpr (FMT == kKvFmtNvfp4) {
#pragma unroll
    for (uint32_t i = 0; i < Cfg::kBlockScales; i += 512) {
      const uint32_t o = i + lane * 16;
      const int r = o / (D / 16), row = at.row(t, r);
      if (o < Cfg::kBlockScales)
        ts_copy16_or_zeros(blocks + o, from.block_scales + static_cast<int64_t>(max(row, 0) + (r & in_box)) * (D / 16),
                           row >= 0);
    }
  }
#pragma unroll
  for (int i = 0; i < TILE; i += 128) {
    const int r = i + lane * 4, row = at.row(t, r);
    if (r < TILE) ts_copy16_or_zeros(rows + r * 4, from.row_scales + max(row, 0) + (r & in_box), row >= 0);
  }
}

// ---------------------------------------------------------------- the streaming kernel
// PAGED: a tile comes in boxes, each from its own page, to the places that a whole
// tile's copy would bring it; 16-position slices of pages that are not there (their
// boxes come in as zeros) are left out.
template <int D, int FMT, int NG, int NW, int SLICES, bool PAGED = false>
__global__ void __launch_bounds__((NW + (PAGED ? 8 : 4)) * 32, 1)
    tree_stream_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const TreeStreamParams p) {
  using Cfg = TsCfg<D, FMT, NG, NW, SLICES, kTsTile<FMT>, PAGED>;
  constexpr int KS = D / 16;  // MMA steps of K Q^T, 16-element row blocks of O^T
  constexpr bool kQuant = FMT != kKvFmtBf16;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // Pointer arithmetic, not an integer round trip: the compiler then knows that
  // what it points to is shared memory.
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // Joining buffers: o [warp][row][kJoinStride], then m [warp][row] and l [warp][row].
  auto join_o = [&](int i) { return reinterpret_cast<float*>(smem + Cfg::kOffComb + i * (Cfg::kComb / Cfg::kJoins)); };
  auto join_m = [&](int i) { return join_o(i) + Cfg::kJoinO / 4; };
  // Element e of row r (of 8 NG): rows in the order that keeps stores of a
  // fragment in different banks, elements of quantised formats rotated in their
  // lane's D / 8 for the same reason.
  auto join_at = [&](int r, int e) {
    constexpr int W = D / 8;
    const int row = (r & ~7) + (r & 1) * 4 + ((r & 7) >> 1);
    const int at = kQuant ? e / W * W + (e % W + 4 * (e / W * W / 32)) % W : e;
    return row * Cfg::kJoinStride + at;
  };
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* empty = full + Cfg::kStages;
  uint64_t* join_full = empty + Cfg::kStages;
  uint64_t* join_free = join_full + Cfg::kJoins;
  int* prefix = reinterpret_cast<int*>(smem + Cfg::kOffPrefix);
  __shared__ volatile unsigned s_bad;  // a wait gave up
  [[maybe_unused]] __shared__ unsigned s_absent[PAGED ? Cfg::kStages : 1];  // slices of a stage that are not there

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  const int rc_n = p.row_chunks, pw_n = NW / rc_n;       // row chunks, position warps per chunk
  constexpr int kTurns = Cfg::kTurns;
  const int groups = pw_n >= kTurns ? pw_n / kTurns : 1; // tiles alternate between groups
  const int units = p.kv_heads * p.passes;
  const int nq = p.group * p.tokens;                     // query rows per KV head

  pdl_launch_dependents();  // the join waits for this kernel's memory itself
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      // K's and V's bytes, and the lanes that copy scales (PAGED: of K and of V by warps of their own)
      mbar_init(&full[s], (PAGED && p.loaders == 4 ? 4 : 2) + (!kQuant ? 0 : PAGED ? 64 : 32));
      mbar_init(&empty[s], pw_n >= kTurns ? kTurns * rc_n : NW);
    }
    for (int i = 0; i < Cfg::kJoins; ++i) {
      mbar_init(&join_full[i], NW);
      mbar_init(&join_free[i], Cfg::kJoiners);
    }
    fence_mbar_init();
    s_bad = 0u;
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
  }
  // Nothing of global memory before this: the launch may overlap the kernel ahead.
  pdl_wait();
  ts_prefix<PAGED>(p, units, kTsTile<FMT>, prefix);
  const int n_tiles = PAGED ? ts_places(p, prefix, units) : prefix[p.batch];
  // With fewer tiles than CTAs only the first n_tiles CTAs take part, so that
  // every CTA between a unit's first and last holds one of its tiles.
  const int G = min(n_tiles, p.grid);
  if (threadIdx.x < 2) p.part_slots[2 * cta + threadIdx.x] = make_int4(-1, 0, 0, 0);
  if (cta >= G) return;
  const int x0 = PAGED ? ts_first_tile_weighted(p, prefix, units, cta, G) : ts_first_tile(n_tiles, cta, G);
  const int x1 = PAGED ? ts_first_tile_weighted(p, prefix, units, cta + 1, G) : ts_first_tile(n_tiles, cta + 1, G);
  __syncthreads();

  // 128 registers a thread at launch: the consumers take what the others give.
  if constexpr (PAGED) {
    if (warp < NW) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTsPagedRegs));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTsPagedOtherRegs));
  }

  if (warp >= NW + Cfg::kLoaders) {
    // ---------------------------------------------------------------- joins: every kJoiners-th row of a segment
    TsWalk w;
    bool more = w.begin(prefix, p.batch, units, x0, x1);
    int buf = 0;
    uint32_t phase = 0;
    for (; more; more = w.next()) {
      const int pass = w.u % p.passes, kvh = w.u / p.passes, n_first = pass * p.rows_per_pass;
      const int rows = min(p.rows_per_pass, nq - n_first);
      [[maybe_unused]] const int tokens = ts_tokens<PAGED>(p, w.b);
      const bool whole = w.t0 == 0 && w.t1 == w.nt;
      const int64_t slot = 2 * static_cast<int64_t>(cta) + (w.x == x0 ? 0 : 1);
      if (!whole && warp == NW + Cfg::kLoaders && lane == 0) ts_write_slot<PAGED>(p, n_tiles, G, cta, x0, w);
      if (!__all_sync(kFull, ts_wait(&join_full[buf], phase, &s_bad))) return;
      const float *so = join_o(buf), *sm_m = join_m(buf), *sm_l = sm_m + NW * Cfg::kRows;
      for (int r = warp - NW - Cfg::kLoaders; r < rows; r += Cfg::kJoiners) {
        // Position warp `lane` of the row's chunk: its factor.
        const int chunk = r / Cfg::kRows, rr = r % Cfg::kRows;
        const int at = (lane * rc_n + chunk) * Cfg::kRows + rr;
        const float mu = lane < pw_n ? sm_m[at] : -INFINITY, lu = lane < pw_n ? sm_l[at] : 0.0f;
        const float mx = warp_max_f32(mu);
        const float fu = mu == -INFINITY ? (lu == 0.0f ? 0.0f : 1.0f) : ts_exp2(mu - mx);
        const float l = warp_sum_f32(lu * fu), inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
        const int n = n_first + r;
        [[maybe_unused]] const bool padding = PAGED && n / p.group >= tokens;
        const int64_t out = static_cast<int64_t>((w.b * p.tokens + n / p.group) * p.q_heads + kvh * p.group + n % p.group) * D;
#pragma unroll
        for (int e = 2 * lane; e < D; e += 64) {
          float2 o = make_float2(0.0f, 0.0f);
          for (int u = 0; u < pw_n; ++u) {
            const float f = __shfl_sync(kFull, fu, u);
            const float2 v = *reinterpret_cast<const float2*>(so + (u * rc_n + chunk) * Cfg::kRows * Cfg::kJoinStride + join_at(rr, e));
            o.x = f == 0.0f ? o.x : fmaf(v.x, f, o.x);
            o.y = f == 0.0f ? o.y : fmaf(v.y, f, o.y);
          }
          if (whole)
            *reinterpret_cast<uint32_t*>(p.ctx + out + e) =
                l == 0.0f || padding ? 0u : ts_pack_bf16(o.x * inv, o.y * inv);
          else
            *reinterpret_cast<float2*>(p.part_o + (slot * p.rows_per_pass + r) * D + e) = o;
        }
        if (!whole && lane == 0) p.part_ml[slot * p.rows_per_pass + r] = make_float2(mx, l);
      }
      __syncwarp();
      if (lane == 0) ts_arrive(&join_free[buf]);
      if (++buf == Cfg::kJoins) {
        buf = 0;
        phase ^= 1u;
      }
    }
    return;
  }

  if (warp >= NW) {
    // ---------------------------------------------------------------- loads: warp NW K, the next one V and scales
    // (PAGED: two warps K, two V)
    // Scales go by 16-byte copies of a whole warp: a bulk copy takes one thread over a hundred cycles to
    // issue, and four of them per tile held E4M3 and NVFP4 caches at 0.8 and 0.4 of the HBM rate.
    const bool is_v = PAGED ? warp >= NW + 2 : warp > NW;
    // PAGED: with four loaders this warp's every other box, the scales for the second; with two all of it.
    [[maybe_unused]] const int split = PAGED && p.loaders == 4 ? 1 : 0, half = (warp - NW) & 1;
    if (PAGED && half > split) return;
    if (!PAGED && lane != 0 && !(is_v && kQuant)) return;
    TsWalk w;
    bool more = w.begin(prefix, p.batch, units, x0, x1);
    int stage = 0;
    uint32_t phase = 0;
    [[maybe_unused]] const int64_t all_rows = static_cast<int64_t>(p.batch) * p.kv_heads * p.capacity;
    [[maybe_unused]] TsBoxes<kTsTile<FMT>> at;
    int filled = 0;  // stages, from the first tile on
    bool ok = true;
    while (more && ok) {
      const int64_t row0 = (static_cast<int64_t>(w.b) * p.kv_heads + w.u / p.passes) * p.capacity;
      if constexpr (PAGED) at.begin(p, w.b, w.u / p.passes, ts_lengths(p, prefix)[w.b].y, w.t0, w.t1, lane);
      for (int t = w.t0; t < w.t1; ++t) {
        ok = filled < Cfg::kStages || ts_wait(&empty[stage], phase ^ 1u, &s_bad);
        if constexpr (PAGED) ok = __all_sync(kFull, ok);
        if (!ok) break;
        uint8_t* st = smem + stage * Cfg::kStage;
        const int64_t row = row0 + static_cast<int64_t>(t) * kTsTile<FMT>;
        if constexpr (PAGED) {
          at.advance(p, t, lane);
          const int of_slice = at.row(t, lane * 16);  // lane i's 16-position slice
          const unsigned absent = __ballot_sync(kFull, lane < kTsTile<FMT> / 16 && of_slice < 0);
          if (lane == 0 && !is_v && !half) s_absent[stage] = absent;
          // Lane i's box, of this warp's.  A thread takes some 200 cycles to issue a copy, whatever its size: with
          // one warp each for K and V pages of 16 held E4M3 at 111 us where whole tiles took 102 (NVFP4 111, 94).
          const int box = (lane << split) + half, mine = at.row(t, box << p.box_log2);
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], Cfg::kCodes >> split);
          __syncwarp();
          if (box < 1 << at.per_log2) {
            // Behind the pool's last row: zeros.
            const int from = mine >= 0 ? mine : p.pg.pages * p.kv_heads * p.pg.page_size;
            uint8_t* dst = st + (is_v ? Cfg::kOffV : 0);
            const CUtensorMap* map = is_v ? &tm_v : &tm_k;
            if constexpr (!kQuant) {
#pragma unroll
              for (int bx = 0; bx < D / 64; ++bx)
                ts_tma_2d(dst + bx * (kTsTile<FMT> * 128) + (box << p.box_log2) * 128, map, bx * 64, from, &full[stage]);
            } else {  // rows stand in groups of 16
              ts_tma_2d(dst + (box << p.box_log2) * Cfg::kRowBytes, map, 0, from / 16 * (16 * Cfg::kRowBytes / 128),
                        &full[stage]);
            }
          }
          __syncwarp();
        } else if (lane == 0) {
          uint8_t* dst = st + (is_v ? Cfg::kOffV : 0);
          const CUtensorMap* map = is_v ? &tm_v : &tm_k;
          mbar_arrive_expect_tx(&full[stage], Cfg::kCodes);
          if constexpr (!kQuant) {
#pragma unroll
            for (int bx = 0; bx < D / 64; ++bx)
              ts_tma_2d(dst + bx * (kTsTile<FMT> * 128), map, bx * 64, static_cast<int>(row), &full[stage]);
          } else {  // the codes as a matrix of 128-byte lines
            ts_tma_2d(dst, map, 0, static_cast<int>(row * Cfg::kRowBytes / 128), &full[stage]);
          }
        }
        if constexpr (kQuant && PAGED) {
          if (half == split) {
            ts_load_scales_paged<D, FMT, Cfg, kTsTile<FMT>>(st + (is_v ? Cfg::kOffVb : Cfg::kOffKb),
                                                            st + (is_v ? Cfg::kOffVr : Cfg::kOffKr), is_v ? p.v : p.k, at,
                                                            t, lane);
            ts_copy_arrive(&full[stage]);
          }
        } else if constexpr (kQuant) {
          if (is_v) {
            ts_load_scales<D, FMT, Cfg, kTsTile<FMT>>(st, p, row, all_rows, lane);
            ts_copy_arrive(&full[stage]);
          }
        }
        ++filled;
        if (++stage == Cfg::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      more = w.next();
    }
    if constexpr (kQuant) ts_copies_landed();
    if (lane == 0) ts_all_landed<Cfg::kStages>(full, filled);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int g = lane >> 2, tq = lane & 3;  // fragment row / column pair
  const int rc = warp % rc_n, pw = warp / rc_n;
  const int turns = pw_n >= kTurns ? 1 : kTurns / pw_n;  // per tile and warp
  const int turn0 = pw_n >= kTurns ? pw % kTurns : pw * turns;
  TsWalk w;
  bool more = w.begin(prefix, p.batch, units, x0, x1);
  const int warp_slot = pw * rc_n + rc;
  int join = 0;
  uint32_t join_phase = 0;
  int stage = 0, turn = 0;  // the CTA's tile counter modulo kStages, modulo groups
  uint32_t phase = 0;
  while (more) {
    const int b = w.b, kvh = w.u / p.passes, pass = w.u % p.passes;
    const int past = PAGED ? ts_lengths(p, prefix)[b].x : ts_past(p, b);
    const int vis = PAGED ? ts_lengths(p, prefix)[b].y : ts_visible(p, b);
    const int n0 = pass * p.rows_per_pass + rc * Cfg::kRows;  // this warp's first query row
    // Query row n = t * group + j; global row of q and ctx:
    auto q_row = [&](int n) -> int64_t {
      return (b * p.tokens + n / p.group) * p.q_heads + kvh * p.group + n % p.group;
    };

    // ---- Q^T fragments: this lane's column is n0 + 8 j + g; q_scale: of its score columns 2 tq, 2 tq + 1
    uint32_t qb[NG][KS][2];
    float q_scale[NG][2];
    int tok[NG][2];  // drafted token of the score columns (-1: no such row)
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int n = n0 + 8 * j + g;
      const uint16_t* src = p.q + q_row(n < nq ? n : 0) * D;
      float own = 1.0f;
      if constexpr (!kQuant) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qb[j][ks][0] = n < nq ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * tq) : 0u;
          qb[j][ks][1] = n < nq ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + 2 * tq) : 0u;
        }
      } else {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint2 e = n < nq ? *reinterpret_cast<const uint2*>(src + (D / 4) * tq + 4 * ks) : make_uint2(0u, 0u);
          qb[j][ks][0] = e.x;
          qb[j][ks][1] = e.y;
          top = max(top, max(max(e.x & 0x7fffu, (e.x >> 16) & 0x7fffu), max(e.y & 0x7fffu, (e.y >> 16) & 0x7fffu)));
        }
        top = max(top, __shfl_xor_sync(kFull, top, 1));
        top = max(top, __shfl_xor_sync(kFull, top, 2));
        // 2^e that brings the row's largest element to [2^14, 2^15)
        const int ex = static_cast<int>(top >> 7);
        const int e = (ex == 0 || ex == 255) ? 0 : min(14 - (ex - 127), 100);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        own = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t e2 = qb[j][ks][i];
            qb[j][ks][i] = ts_pack_f16(__uint_as_float(e2 << 16) * up, __uint_as_float(e2 & 0xffff0000u) * up);
          }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        q_scale[j][c] = __shfl_sync(kFull, own, (2 * tq + c) * 4) * p.scale_log2;
        const int col = n0 + 8 * j + 2 * tq + c;
        tok[j][c] = col < nq ? col / p.group : -1;
      }
    }

    float m_run[NG][2], l_run[NG][2], acc[NG][KS][4];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      m_run[j][0] = m_run[j][1] = -INFINITY;
      l_run[j][0] = l_run[j][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < KS; ++i) acc[j][i][0] = acc[j][i][1] = acc[j][i][2] = acc[j][i][3] = 0.0f;
    }
    float g_run[NG][2], p_unit[NG][2];  // G of the score columns, 2^5 / G
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      g_run[j][0] = g_run[j][1] = kTsMinUnit;
      p_unit[j][0] = p_unit[j][1] = kTsPScale / kTsMinUnit;
    }

    // SL slices of 16 positions of the tile in `st`, first position pos0 (row r0 of the tile).
    auto slice = [&](auto edge_tag, auto slices_tag, const uint8_t* st, int r0, int pos0) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      constexpr int SL = decltype(slices_tag)::value;
      const uint8_t *kt = st, *vt = st + Cfg::kOffV;
      // ---- S^T = K Q^T of one slice; score rows: its positions g and 8 + g
      auto scores = [&](int r0, float (&s)[NG][2][4]) {  // two accumulators, alternate steps
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[j][h][0] = s[j][h][1] = s[j][h][2] = s[j][h][3] = 0.0f;
      if constexpr (FMT == kKvFmtBf16) {
        const int mat = lane >> 3, r = r0 + (mat & 1) * 8 + (lane & 7);
        const uint32_t base = smem_u32(kt) + r * 128;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int c = (ks & 3) * 2 + (mat >> 1);
          uint32_t a[4];
          ts_ldsm4(base + (ks >> 2) * (kTsTile<FMT> * 128) + ((c ^ (lane & 7)) << 4), a);
#pragma unroll
          for (int j = 0; j < NG; ++j) ts_mma<FMT>(s[j][ks & 1], a[0], a[1], a[2], a[3], qb[j][ks][0], qb[j][ks][1]);
        }
      } else if constexpr (FMT == kKvFmtE4m3) {
        // D / 4 codes per row and lane, four per MMA step
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint32_t o = (D / 4) * tq + 16 * i;
          const uint4 w0 = *reinterpret_cast<const uint4*>(kt + ts_swz((r0 + g) * D + o));
          const uint4 w1 = *reinterpret_cast<const uint4*>(kt + ts_swz((r0 + 8 + g) * D + o));
          const uint32_t c0[4] = {w0.x, w0.y, w0.z, w0.w}, c1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a0, a1, a2, a3;
            ts_e4m3x4(c0[e], a0, a2);
            ts_e4m3x4(c1[e], a1, a3);
            const int ks = 4 * i + e;
#pragma unroll
            for (int j = 0; j < NG; ++j) ts_mma<FMT>(s[j][ks & 1], a0, a1, a2, a3, qb[j][ks][0], qb[j][ks][1]);
          }
        }
      } else {
        // D / 4 codes per row and lane: words of eight, two MMA steps each; a block scale per two words
        constexpr int NWORD = D / 32, NB = D / 64;
        const uint8_t* kb = st + Cfg::kOffKb;
        uint32_t c[2][NWORD], bs[2][NB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = r0 + 8 * h + g;
          if constexpr (D == 64) {
            const uint2 v = *reinterpret_cast<const uint2*>(kt + ts_swz(r * (D / 2) + (D / 8) * tq));
            c[h][0] = v.x;
            c[h][1] = v.y;
            bs[h][0] = kb[r * (D / 16) + tq];
          } else {
#pragma unroll
            for (int i = 0; i < NWORD / 4; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(kt + ts_swz(r * (D / 2) + (D / 8) * tq + 16 * i));
              c[h][4 * i] = v.x;
              c[h][4 * i + 1] = v.y;
              c[h][4 * i + 2] = v.z;
              c[h][4 * i + 3] = v.w;
              const uint32_t two = *reinterpret_cast<const uint16_t*>(kb + r * (D / 16) + NB * tq + 2 * i);
              bs[h][2 * i] = two & 0xffu;
              bs[h][2 * i + 1] = two >> 8;
            }
          }
#pragma unroll
          for (int i = 0; i < NB; ++i) bs[h][i] = e4m3x2_to_f16x2(bs[h][i] * 0x101u);  // in both halves
        }
#pragma unroll
        for (int i = 0; i < NWORD; ++i) {
          uint32_t d0[4], d1[4];
          e2m1x8_to_f16x2x4(c[0][i], d0);
          e2m1x8_to_f16x2x4(c[1][i], d1);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d0[e] = ts_hmul2(d0[e], bs[0][i / 2]);
            d1[e] = ts_hmul2(d1[e], bs[1][i / 2]);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int ks = 2 * i + e;
#pragma unroll
            for (int j = 0; j < NG; ++j)
              ts_mma<FMT>(s[j][e], d0[2 * e], d1[2 * e], d0[2 * e + 1], d1[2 * e + 1], qb[j][ks][0], qb[j][ks][1]);
          }
        }
      }

      };
      float s[SL][NG][2][4];
#pragma unroll
      for (int z = 0; z < SL; ++z) scores(r0 + 16 * z, s[z]);

      // ---- scores in log2 units; sc[z][j][i]: position pos0 + 16 z + g (+ 8 for i >= 2), column 2 tq + (i & 1)
      [[maybe_unused]] float k_unit[SL][2], v_unit[SL][2];
      if constexpr (kQuant) {
#pragma unroll
        for (int z = 0; z < SL; ++z)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = r0 + 16 * z + 8 * h + g;
            k_unit[z][h] = reinterpret_cast<const float*>(st + Cfg::kOffKr)[r];
            v_unit[z][h] = reinterpret_cast<const float*>(st + Cfg::kOffVr)[r];
          }
      }
      float sc[SL][NG][4];
      bool sees[SL][NG][4];
      bool above = false;
#pragma unroll
      for (int z = 0; z < SL; ++z)
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = (s[z][j][0][i] + s[z][j][1][i]) * q_scale[j][i & 1];
            if constexpr (kQuant) x *= k_unit[z][i >> 1];
            if constexpr (EDGE) {
              const int pos = pos0 + 16 * z + g + (i >> 1) * 8, u = pos - past;
              const int t = tok[j][i & 1];
              bool ok = t >= 0 && pos < vis;
              if (ok && u >= 0)
                ok = p.mask ? p.mask[b * p.mask_stride + static_cast<int64_t>(t) * p.tokens + u] != 0 : u <= t;
              sees[z][j][i] = ok;
              if (!ok) x = -INFINITY;
            } else {
              sees[z][j][i] = true;
            }
            sc[z][j][i] = x;
            above |= x > m_run[j][i & 1] + kTsSlack<FMT>;
          }
      auto rescale = [&](const float (&f)[NG][2]) {
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            acc[j][i][0] *= f[j][0];
            acc[j][i][1] *= f[j][1];
            acc[j][i][2] *= f[j][0];
            acc[j][i][3] *= f[j][1];
          }
      };
      // ---- the reference moves (for every column) when a score passes it by the slack
      if (__any_sync(kFull, above)) {
        float alpha[NG][2];
        [[maybe_unused]] bool low = false;
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(sc[0][j][c], sc[0][j][c + 2]);
#pragma unroll
            for (int z = 1; z < SL; ++z) mx = fmaxf(mx, fmaxf(sc[z][j][c], sc[z][j][c + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
            const float m_new = fmaxf(m_run[j][c], mx + kTsLift<FMT>);
            const bool fresh = m_run[j][c] == -INFINITY;
            alpha[j][c] = fresh ? 0.0f : ts_exp2(m_run[j][c] - m_new);
            m_run[j][c] = m_new;
            l_run[j][c] *= alpha[j][c];
            if constexpr (kQuant) {  // G shrinks as what the accumulators stand for does, down to its least
              const float g = fresh ? kTsMinUnit : g_run[j][c] * alpha[j][c];
              alpha[j][c] = g < kTsMinUnit ? __fdiv_rn(g, kTsMinUnit) : 1.0f;
              low |= g < kTsMinUnit;
              g_run[j][c] = fmaxf(g, kTsMinUnit);
              p_unit[j][c] = __fdiv_rn(kTsPScale, g_run[j][c]);
            }
          }
        if (!kQuant || __any_sync(kFull, low)) rescale(alpha);
      }
      float pr[SL][NG][4];
#pragma unroll
      for (int z = 0; z < SL; ++z)
#pragma unroll
        for (int j = 0; j < NG; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i)  // -inf only stands for a key that is not seen, or one that weighs nothing
            pr[z][j][i] = sc[z][j][i] == -INFINITY ? 0.0f : ts_exp2(sc[z][j][i] - m_run[j][i & 1]);
          l_run[j][0] += pr[z][j][0] + pr[z][j][2];
          l_run[j][1] += pr[z][j][1] + pr[z][j][3];
        }
      // ---- P^T as B fragments
      uint32_t ph[SL][NG][2];
      [[maybe_unused]] uint32_t pl[SL][NG][2];  // second term, BF16 only
      if constexpr (kQuant) {
        float con[SL][NG][4];  // contributions p_j gamma_j
#pragma unroll
        for (int z = 0; z < SL; ++z)
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              con[z][j][i] = pr[z][j][i] * v_unit[z][i >> 1];
              if constexpr (EDGE)  // a row that is not seen may have any scale
                if (!sees[z][j][i]) con[z][j][i] = 0.0f;
            }
        uint32_t top = 0u;
        auto pack = [&] {
#pragma unroll
          for (int z = 0; z < SL; ++z)
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                ph[z][j][i] = ts_pack_f16(con[z][j][2 * i] * p_unit[j][0], con[z][j][2 * i + 1] * p_unit[j][1]);
                top = ts_largest(top, ph[z][j][i]);
              }
        };
        pack();
        // G up to the largest finite contribution where one has passed it by the slack
        if (__any_sync(kFull, max(top & 0x7fffu, top >> 16 & 0x7fffu) >= kTsPLimit)) {
          float f[NG][2];
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = 0.0f;
#pragma unroll
              for (int z = 0; z < SL; ++z)
#pragma unroll
                for (int i = c; i < 4; i += 2) {
                  const float size = fabsf(con[z][j][i]);
                  if (size < INFINITY) mx = fmaxf(mx, size);
                }
              mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
              mx = fmaxf(mx, g_run[j][c]);
              f[j][c] = __fdiv_rn(g_run[j][c], mx);
              g_run[j][c] = mx;
              p_unit[j][c] = __fdiv_rn(kTsPScale, mx);
            }
          rescale(f);
          pack();
        }
#pragma unroll
        for (int z = 0; z < SL; ++z)
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) ph[z][j][i] = ts_transpose(ph[z][j][i]);
      } else {
#pragma unroll
        for (int z = 0; z < SL; ++z)
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float wt[2];
#pragma unroll
              for (int c = 0; c < 2; ++c)
                wt[c] = EDGE && !sees[z][j][2 * i + c] ? 0.0f : pr[z][j][2 * i + c];
              const uint32_t h = ts_pack_bf16(wt[0], wt[1]);
              ph[z][j][i] = ts_transpose(h);
              pl[z][j][i] =
                  ts_transpose(ts_pack_bf16(wt[0] - __uint_as_float(h << 16), wt[1] - __uint_as_float(h & 0xffff0000u)));
            }
      }
      // ---- O^T += V^T P^T of one slice
      auto output = [&](int r0, int pos0, const uint32_t (&ph)[NG][2], [[maybe_unused]] const uint32_t (&pl)[NG][2],
                        [[maybe_unused]] const float (&pr)[NG][4], [[maybe_unused]] const bool (&sees)[NG][4]) {
      uint32_t bad = 0;  // positions (bits) whose V holds an infinity or NaN somewhere in this lane's part
      // Positions of the fragments' halves: 2 tq, 2 tq + 1 (registers 0, 1) and + 8 (registers 2, 3).
      auto clean = [&](uint32_t (&a)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pos = pos0 + 2 * tq + (i >> 1) * 8;
          if (pos >= vis) a[i] = 0u;
          else if (pos + 1 >= vis) a[i] &= 0x0000ffffu;
          uint32_t two = 0;
          a[i] = ts_finite<FMT>(a[i], two);
          bad |= two << (2 * tq + (i >> 1) * 8);
        }
      };
      auto pv = [&](int mt, uint32_t (&a)[4]) {
        if constexpr (EDGE) clean(a);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          ts_mma<FMT>(acc[j][mt], a[0], a[1], a[2], a[3], ph[j][0], ph[j][1]);
          if constexpr (!kQuant) ts_mma<FMT>(acc[j][mt], a[0], a[1], a[2], a[3], pl[j][0], pl[j][1]);
        }
      };
      if constexpr (FMT == kKvFmtBf16) {
        const int mat = lane >> 3, r = r0 + (mat >> 1) * 8 + (lane & 7);
        const uint32_t base = smem_u32(vt) + r * 128;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          const int c = (mt & 3) * 2 + (mat & 1);
          uint32_t a[4];
          ts_ldsm4_trans(base + (mt >> 2) * (kTsTile<FMT> * 128) + ((c ^ (lane & 7)) << 4), a);
          pv(mt, a);
        }
      } else {
        // D / 8 codes of four positions per lane; row g of block mt is element D/8 g + 2 mt, row g + 8 the next
        constexpr int BYTES = Cfg::kRowBytes / 8;  // 4 to 32
        uint32_t c[4][BYTES / 4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + 2 * tq + (e & 1) + (e >> 1) * 8;
          const uint32_t o = r * Cfg::kRowBytes + BYTES * g;
          if constexpr (BYTES == 4) {
            c[e][0] = *reinterpret_cast<const uint32_t*>(vt + ts_swz(o));
          } else if constexpr (BYTES == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(vt + ts_swz(o));
            c[e][0] = v.x;
            c[e][1] = v.y;
          } else {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(vt + ts_swz(o + 16 * i));
              c[e][4 * i] = v.x;
              c[e][4 * i + 1] = v.y;
              c[e][4 * i + 2] = v.z;
              c[e][4 * i + 3] = v.w;
            }
          }
        }
        if constexpr (FMT == kKvFmtE4m3) {
#pragma unroll
          for (int i = 0; i < BYTES / 4; ++i) {
            // Two positions' codes of an element side by side before they are decoded: half of the permutations.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h ? 0x7362 : 0x5140;
              uint32_t a[4];
              ts_e4m3x4(__byte_perm(c[0][i], c[1][i], sel), a[0], a[1]);
              ts_e4m3x4(__byte_perm(c[2][i], c[3][i], sel), a[2], a[3]);
              pv(2 * i + h, a);
            }
          }
        } else {
          constexpr int NB = D == 256 ? 2 : 1;  // block scales per lane and position
          const uint8_t* vb = st + Cfg::kOffVb;
          uint32_t bs[NB][2];  // [block][positions 2 tq and + 1, + 8 and + 9]
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint8_t* at = vb + (r0 + 2 * tq + 8 * h) * (D / 16) + (D / 8 * g + 16 * i) / 16;
              bs[i][h] = e4m3x2_to_f16x2(at[0] | (static_cast<uint32_t>(at[D / 16]) << 8));
            }
#pragma unroll
          for (int i = 0; i < BYTES / 4; ++i) {
            // Two positions' codes of an element side by side before they are decoded; even and odd elements.
            uint32_t d[2][2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = c[2 * e][i], y = c[2 * e + 1][i];
              e2m1x8_to_f16x2x4((x & 0x0f0f0f0fu) | (y << 4 & 0xf0f0f0f0u), d[e][0]);
              e2m1x8_to_f16x2x4((x >> 4 & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), d[e][1]);
            }
            const uint32_t b0 = bs[i * NB / (BYTES / 4)][0], b1 = bs[i * NB / (BYTES / 4)][1];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              uint32_t a[4] = {ts_hmul2(d[0][0][h], b0), ts_hmul2(d[0][1][h], b0), ts_hmul2(d[1][0][h], b1),
                               ts_hmul2(d[1][1][h], b1)};
              pv(4 * i + h, a);
            }
          }
        }
      }
      if constexpr (EDGE) {
        // Infinities and NaN of V that were zeroed: added for the queries that see the row.
        bad = __reduce_or_sync(kFull, bad);
        while (bad) {
          const int r = __ffs(bad) - 1;
          bad &= bad - 1;
          const int from = (r & 7) * 4 + tq;
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float lo = __shfl_sync(kFull, sees[j][c] ? pr[j][c] : -1.0f, from);
              const float hi = __shfl_sync(kFull, sees[j][c + 2] ? pr[j][c + 2] : -1.0f, from);
              const float pj = r < 8 ? lo : hi;
              if (!(pj < 0.0f)) {
#pragma unroll
                for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const int d = FMT == kKvFmtBf16 ? 16 * mt + 8 * h + g : D / 8 * g + 2 * mt + h;
                    const float x = ts_v_element<D, FMT>(vt, st + Cfg::kOffVb, r0 + r, d);
                    if (!isfinite(x)) acc[j][mt][2 * h + c] += pj * x;
                  }
              }
            }
        }
      }
      };
#pragma unroll
      for (int z = 0; z < SL; ++z) output(r0 + 16 * z, pos0 + 16 * z, ph[z], pl[z], pr[z], sees[z]);
    };

    for (int t = w.t0; t < w.t1; ++t) {
      const bool mine = pw_n < kTurns || turn == pw / kTurns;
      if (mine) {
        if (!__all_sync(kFull, ts_wait(&full[stage], phase, &s_bad))) return;
        const uint8_t* st = smem + stage * Cfg::kStage;
        unsigned absent = 0u;
        if constexpr (PAGED) absent = s_absent[stage];
        for (int i = 0; i < turns; ++i) {
          const int r0 = (turn0 + i) * 16 * SLICES;
          const int pos0 = t * kTsTile<FMT> + r0;
          if (pos0 >= vis || (PAGED && n0 >= nq)) break;
          const unsigned gone = absent >> (r0 / 16) & ((1u << SLICES) - 1u);  // slices whose page is not there
          using Slices = std::integral_constant<int, SLICES>;
          if (pos0 + 16 * SLICES <= past && !gone) {
            slice(std::false_type{}, Slices{}, st, r0, pos0);
          } else if constexpr (PAGED) {  // one at a time: half of the code that a segment's end has to fetch
#pragma unroll 1
            for (int z = 0; z < SLICES; ++z)
              if (pos0 + 16 * z < vis && !(gone >> z & 1u))
                slice(std::true_type{}, std::integral_constant<int, 1>{}, st, r0 + 16 * z, pos0 + 16 * z);
          } else {
            slice(std::true_type{}, Slices{}, st, r0, pos0);
          }
        }
        __syncwarp();
        if (lane == 0) ts_arrive(&empty[stage]);
      }
      if (++turn == groups) turn = 0;
      if (++stage == Cfg::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }

    // ---- this segment's (m, l, o) to the joining warps
    if (!__all_sync(kFull, ts_wait(&join_free[join], join_phase ^ 1u, &s_bad))) return;
    float *so = join_o(join), *sm_m = join_m(join), *sm_l = sm_m + NW * Cfg::kRows;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float unit = kQuant ? g_run[j][c] * (1.0f / kTsPScale) : 1.0f;
        float l = l_run[j][c];
        l += __shfl_xor_sync(kFull, l, 4);
        l += __shfl_xor_sync(kFull, l, 8);
        l += __shfl_xor_sync(kFull, l, 16);
        const int r = 8 * j + 2 * tq + c;
        if (g == 0) {
          sm_m[warp_slot * Cfg::kRows + r] = m_run[j][c];
          sm_l[warp_slot * Cfg::kRows + r] = l;
        }
        float* o = so + warp_slot * Cfg::kRows * Cfg::kJoinStride;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          if constexpr (kQuant) {
            *reinterpret_cast<float2*>(o + join_at(r, D / 8 * g + 2 * mt)) =
                make_float2(acc[j][mt][c] * unit, acc[j][mt][2 + c] * unit);
          } else {
            o[join_at(r, 16 * mt + g)] = acc[j][mt][c];
            o[join_at(r, 16 * mt + 8 + g)] = acc[j][mt][2 + c];
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) ts_arrive(&join_full[join]);
    if (++join == Cfg::kJoins) {
      join = 0;
      join_phase ^= 1u;
    }
    more = w.next();
  }
}

// ---------------------------------------------------------------- joining partials
// Grid (slot, group of rows): a warp joins one query row of a unit that several
// CTAs share, in CTA order.  Only the slot of the unit's first part has work.
constexpr int kTsJoinWarps = 8;

template <int D, bool PAGED = false>
__global__ void __launch_bounds__(kTsJoinWarps * 32) tree_stream_combine_kernel(const TreeStreamParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int4 unit = __ldcg(&p.part_slots[blockIdx.x]);
  if (unit.x < 0) return;
  const int b = unit.x, u = unit.y, c0 = unit.z, c1 = unit.w;
  const int lane = threadIdx.x & 31, r = blockIdx.y * kTsJoinWarps + (threadIdx.x >> 5);
  const int pass = u % p.passes, kvh = u / p.passes, n = pass * p.rows_per_pass + r;
  if (r >= p.rows_per_pass || n >= p.group * p.tokens) return;
  // The unit's part in its first CTA is in this slot, in the others in their first.
  auto at = [&](int c) {
    return (c == c0 ? static_cast<int64_t>(blockIdx.x) : 2 * static_cast<int64_t>(c)) * p.rows_per_pass + r;
  };
  constexpr int V = D / 32;  // elements per lane
  constexpr int kAtOnce = 8;  // parts whose loads are in flight together
  float x[kAtOnce][V];
  auto fetch = [&](int c) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (c + i > c1) break;
      const float* src = p.part_o + at(c + i) * D + lane * V;
      if constexpr (V == 2) {
        *reinterpret_cast<float2*>(x[i]) = __ldcg(reinterpret_cast<const float2*>(src));
      } else {
#pragma unroll
        for (int k = 0; k < V / 4; ++k) reinterpret_cast<float4*>(x[i])[k] = __ldcg(reinterpret_cast<const float4*>(src) + k);
      }
    }
  };
  fetch(c0);  // beside the (m, l) loads
  float mx = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, __ldcg(&p.part_ml[at(c)]).x);
  mx = warp_max_f32(mx);
  float o[V] = {}, l = 0.0f;
  for (int base = c0; base <= c1; base += 32) {
    const float2 ml = base + lane <= c1 ? __ldcg(&p.part_ml[at(base + lane)]) : make_float2(-INFINITY, 0.0f);
    const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ts_exp2(ml.x - mx);
    l = fmaf(ml.y, f, l);
    const int end = min(base + 31, c1);
    for (int c = base; c <= end; c += kAtOnce) {
      if (c != c0) fetch(c);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float fc = __shfl_sync(kFull, f, (c - base + i) & 31);
        if (c + i > c1 || fc == 0.0f) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = fmaf(x[i][k], fc, o[k]);
      }
    }
  }
  l = warp_sum_f32(l);
  const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
  const int64_t row = (static_cast<int64_t>(b) * p.tokens + n / p.group) * p.q_heads +
                      static_cast<int64_t>(kvh) * p.group + n % p.group;
  const bool none = l == 0.0f || (PAGED && n / p.group >= ts_tokens<PAGED>(p, b));
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.ctx + row * D + lane * V);
#pragma unroll
  for (int i = 0; i < V / 2; ++i)
    dst[i] = none ? 0u : ts_pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
}

// The same where there are many rows of few parts: a warp joins four rows, eight
// lanes working out one row's weights (eight parts at a time).  With a row per
// warp the divisions, shuffles and address arithmetic of a row were most of the
// instructions, which bound the kernel.
constexpr int kTsJoinRows = 4;

template <int D, bool PAGED = false>
__global__ void __launch_bounds__(kTsJoinWarps * 32) tree_stream_combine4_kernel(const TreeStreamParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int4 unit = __ldcg(&p.part_slots[blockIdx.x]);
  if (unit.x < 0) return;
  const int b = unit.x, u = unit.y, c0 = unit.z, c1 = unit.w;
  const int pass = p.passes == 1 ? 0 : u % p.passes, kvh = p.passes == 1 ? u : u / p.passes;
  const int lane = threadIdx.x & 31, sub = lane & 7, mine = lane >> 3;  // part and row this lane weighs
  const int r0 = (blockIdx.y * kTsJoinWarps + (threadIdx.x >> 5)) * kTsJoinRows;
  const int rows = min(kTsJoinRows, min(p.rows_per_pass, p.group * p.tokens - pass * p.rows_per_pass) - r0);
  if (rows <= 0) return;
  // Row of a part's slot (fewer than 2^31 / D of them): the unit's part in its first CTA is in this slot, in the
  // others in their first.
  auto at = [&](int c) { return (c == c0 ? static_cast<int>(blockIdx.x) : 2 * c) * p.rows_per_pass + r0; };
  constexpr int V = D / 32;  // elements per lane
  float x[2][kTsJoinRows][V];
  auto fetch = [&](int c, float (&y)[kTsJoinRows][V]) {
    const float* src = p.part_o + static_cast<int64_t>(at(c)) * D + lane * V;
#pragma unroll
    for (int i = 0; i < kTsJoinRows; ++i) {
      if (i >= rows) break;
      if constexpr (V == 2) {
        *reinterpret_cast<float2*>(y[i]) = __ldcg(reinterpret_cast<const float2*>(src + i * D));
      } else {
#pragma unroll
        for (int k = 0; k < V / 4; ++k)
          reinterpret_cast<float4*>(y[i])[k] = __ldcg(reinterpret_cast<const float4*>(src + i * D) + k);
      }
    }
  };
  auto stats = [&](int c) {
    return c <= c1 && mine < rows ? __ldcg(&p.part_ml[at(c) + mine]) : make_float2(-INFINITY, 0.0f);
  };
  fetch(c0, x[0]);  // beside the (m, l) loads
  if (c0 < c1) fetch(c0 + 1, x[1]);
  float2 ml = stats(c0 + sub);
  float mx = ml.x;
  for (int c = c0 + 8; c <= c1; c += 8) mx = fmaxf(mx, stats(c + sub).x);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
  float o[kTsJoinRows][V] = {}, l = 0.0f, f = 0.0f;
  auto add = [&](int c, const float (&y)[kTsJoinRows][V]) {
#pragma unroll
    for (int i = 0; i < kTsJoinRows; ++i) {
      const float fc = __shfl_sync(kFull, f, 8 * i + ((c - c0) & 7));
      if (fc == 0.0f) continue;  // uniform; also rows past the last
#pragma unroll
      for (int k = 0; k < V; ++k) o[i][k] = fmaf(y[i][k], fc, o[i][k]);
    }
  };
  for (int c = c0; c <= c1; c += 2) {
    if (((c - c0) & 7) == 0) {
      if (c > c0) ml = stats(c + sub);
      f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ts_exp2(ml.x - mx);
      l = fmaf(ml.y, f, l);
    }
    add(c, x[0]);
    if (c + 2 <= c1) fetch(c + 2, x[0]);
    if (c + 1 <= c1) add(c + 1, x[1]);
    if (c + 3 <= c1) fetch(c + 3, x[1]);
  }
#pragma unroll
  for (int k = 1; k < 8; k <<= 1) l += __shfl_xor_sync(kFull, l, k);
  const int n = pass * p.rows_per_pass + r0 + mine, tok = n / p.group;
  const float inv = l == 0.0f || (PAGED && tok >= ts_tokens<PAGED>(p, b)) ? 0.0f : __fdiv_rn(1.0f, l);
  const int row = (b * p.tokens + tok) * p.q_heads + kvh * p.group + (n - tok * p.group);  // below 2^31
#pragma unroll
  for (int i = 0; i < kTsJoinRows; ++i) {
    if (i >= rows) break;
    const float by = __shfl_sync(kFull, inv, 8 * i);
    const int64_t to = __shfl_sync(kFull, row, 8 * i);
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.ctx + to * D + lane * V);
    uint32_t y[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) y[k] = by == 0.0f ? 0u : ts_pack_bf16(o[i][2 * k] * by, o[i][2 * k + 1] * by);
    if constexpr (V == 2) {
      dst[0] = y[0];
    } else {
#pragma unroll
      for (int k = 0; k < V / 4; ++k) reinterpret_cast<uint2*>(dst)[k] = make_uint2(y[2 * k], y[2 * k + 1]);
    }
  }
}

}  // namespace nvfp4da
