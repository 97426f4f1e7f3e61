// Launches of the streaming and the tensor-core tree attention and their joins, over caches of whole
// sequences and (PAGED) over pools of pages.
#pragma once

#include "kv_host.cuh"
#include "tree_stream.cuh"
#include "tree_tc.cuh"

namespace nvfp4da {

// Adds (or moves, with `clear`) the flags of the paged attention's waits to *flags (paged_capi.cu).
__attribute__((visibility("hidden"))) cudaError_t paged_attention_flags(unsigned* flags, int clear, cudaStream_t s);

namespace {

constexpr int kTsWarps = 8;
// 16-position slices a warp takes at once: two hide the latency of decoding
// codes (E4M3 87 -> 77 us, NVFP4 93 -> 81 us on 8 x 32K positions); BF16 has
// none to hide.
template <int D, int FMT, int NG>
constexpr int ts_slices() { return FMT != kKvFmtBf16 && NG == 1 && D <= 128 ? 2 : 1; }

// Rows from which, and parts a unit has at most (CTAs per unit), where a warp
// joins four rows instead of one: 192 rows over BF16 (16 sequences, 8,000
// positions) 146 -> 141 us in all, 64 rows over NVFP4 (8, 32,000) 159 -> 155;
// with 12 parts a unit the few warps take longer (41 -> 42 us).
constexpr int64_t kJoin4MinRows = 17, kJoin4MaxParts = 8;

template <int D, bool PAGED = false>
cudaError_t launch_tree_combine(const TreeStreamParams& p, cudaStream_t s) {
  const int64_t rows = std::min(p.rows_per_pass, p.group * p.tokens);
  const int64_t units = static_cast<int64_t>(p.batch) * p.kv_heads * p.passes;
  const bool four = rows >= kJoin4MinRows && units * kJoin4MaxParts >= p.grid;
  const dim3 grid(static_cast<unsigned>(2 * p.grid),
                  static_cast<unsigned>(ceil_div(rows, four ? kTsJoinWarps * kTsJoinRows : kTsJoinWarps)));
  return launch(four ? tree_stream_combine4_kernel<D, PAGED> : tree_stream_combine_kernel<D, PAGED>, grid,
                dim3(kTsJoinWarps * 32), 0, s, true, p);
}

template <int D, int FMT, int NG, bool PAGED = false>
cudaError_t launch_tree_stream(const CUtensorMap& tk, const CUtensorMap& tv, const TreeStreamParams& p,
                               cudaStream_t s) {
  constexpr int SL = ts_slices<D, FMT, NG>(), NW = kTsWarps;
  auto* kern = tree_stream_kernel<D, FMT, NG, NW, SL, PAGED>;
  using Cfg = TsCfg<D, FMT, NG, NW, SL, kTsTile<FMT>, PAGED>;
  const uint32_t smem = Cfg::bytes(p.batch);
  if constexpr (PAGED) {  // the warps' register shares are drawn from what the block is launched with
    static const int regs = [&] {
      cudaFuncAttributes a{};
      return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
    }();
    if (regs * Cfg::kThreads < (kTsPagedRegs * NW + kTsPagedOtherRegs * 8) * 32) return cudaErrorLaunchOutOfResources;
  }
  cudaError_t e = ensure_smem(kern, smem);
  if (e != cudaSuccess) return e;
  e = launch(kern, dim3(static_cast<unsigned>(p.grid)), dim3(Cfg::kThreads), smem, s, true, tk, tv, p);
  return e != cudaSuccess ? e : launch_tree_combine<D, PAGED>(p, s);
}

template <int FMT, bool PAGED = false>
cudaError_t launch_tree_stream_d(int64_t head_dim, int wide, const CUtensorMap& tk, const CUtensorMap& tv,
                                 const TreeStreamParams& p, cudaStream_t s) {
  if constexpr (PAGED) {
    switch (head_dim) {
      case 64:
        if constexpr (FMT == kKvFmtE4m3) {  // the others: tcgen05 from 17 rows on
          if (wide == 3) return launch_tree_stream<64, FMT, 3, true>(tk, tv, p, s);
          if (wide == 2) return launch_tree_stream<64, FMT, 2, true>(tk, tv, p, s);
        }
        return launch_tree_stream<64, FMT, 1, true>(tk, tv, p, s);
      case 128: return launch_tree_stream<128, FMT, 1, true>(tk, tv, p, s);
      default: return launch_tree_stream<256, FMT, 1, true>(tk, tv, p, s);
    }
  } else {
    switch (head_dim) {
      case 64:
        return wide == 2 ? launch_tree_stream<64, FMT, 2>(tk, tv, p, s) : launch_tree_stream<64, FMT, 1>(tk, tv, p, s);
      case 128:
        if constexpr (FMT == kKvFmtBf16)  // codes: tcgen05 from 9 rows on
          if (wide == 2) return launch_tree_stream<128, FMT, 2>(tk, tv, p, s);
        return launch_tree_stream<128, FMT, 1>(tk, tv, p, s);
      default: return launch_tree_stream<256, FMT, 1>(tk, tv, p, s);
    }
  }
}

// Query rows per KV head from which tree_tc_kernel runs.  The streaming kernel
// decodes codes in registers for the rows of one warp, this one once for all
// rows.  Both, 8 sequences x 6 KV heads x 4 query heads each, us streaming /
// tcgen05 after 300, 2,000 and 12,000 positions, head_dim 128:
//          8 rows (2 tokens)        12 rows                  20 rows                  64 rows
//   BF16   20/27  23/28  58/69      25/26  30/29   65/69     29/28  37/31   78/72     66/27  78/33  151/75
//   E4M3   20/26  23/33  41/74      22/26  39/32  131/74     26/27  46/35  146/77     47/30  88/38  211/84
//   NVFP4  20/27  24/33  40/72      22/26  38/33  118/72     26/28  45/36  131/77     47/30  87/38  192/82
// and head_dim 64, where a tile is half the bytes and the decoding, but the
// tcgen05 kernel's warps take as long for it:
//          12 rows                  24 rows                  32 rows                  64 rows
//   BF16   27/27  26/28  38/57      22/26  27/26  56/58      27/27  31/26  60/59      41/21  48/27   96/62
//   E4M3   20/23  23/29  45/65      21/24  30/30  62/66      21/24  33/30  66/67      29/25  52/32  106/73
//   NVFP4  20/24  23/30  43/68      20/24  30/31  61/70      21/25  34/31  64/71      29/26  52/32  107/76
constexpr int64_t tc_min_rows(int64_t head_dim, bool bf16) { return head_dim == 64 ? 33 : bf16 ? 13 : 9; }

template <int D, int FMT, bool SPLIT, bool PAGED = false>
cudaError_t launch_tree_tc(const CUtensorMap& tk, const CUtensorMap& tv, const TreeStreamParams& p, cudaStream_t s) {
  auto* kern = tree_tc_kernel<D, FMT, SPLIT, PAGED>;
  const uint32_t smem = TtCfg<D, FMT, SPLIT>::template bytes<PAGED>(p.batch);
  // The warps' register shares are drawn from what the block is launched with.
  static const int regs = [&] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs * kTtThreads < (kTtSoftmaxRegs * kTtSoftmaxWarps + kTtOtherRegs * (kTtThreads / 32 - kTtSoftmaxWarps)) * 32)
    return cudaErrorLaunchOutOfResources;
  cudaError_t e = ensure_smem(kern, smem);
  if (e != cudaSuccess) return e;
  e = launch(kern, dim3(static_cast<unsigned>(p.grid)), dim3(kTtThreads), smem, s, true, tk, tv, p);
  return e != cudaSuccess ? e : launch_tree_combine<D, PAGED>(p, s);
}

template <int FMT, bool PAGED = false>
cudaError_t launch_tree_tc_d(int64_t head_dim, bool split, const CUtensorMap& tk, const CUtensorMap& tv,
                             const TreeStreamParams& p, cudaStream_t s) {
  if (head_dim == 64)
    return split ? launch_tree_tc<64, FMT, true, PAGED>(tk, tv, p, s)
                 : launch_tree_tc<64, FMT, false, PAGED>(tk, tv, p, s);
  return split ? launch_tree_tc<128, FMT, true, PAGED>(tk, tv, p, s)
               : launch_tree_tc<128, FMT, false, PAGED>(tk, tv, p, s);
}

// The tensor map of K or V: BF16 rows in 64-element boxes, codes as 128-byte lines.
bool tree_map(CUtensorMap* map, const nvfp4da_kv_cache& c, const void* base, int64_t tile) {
  const uint64_t rows = static_cast<uint64_t>(c.batch * c.kv_heads * c.capacity), d = c.head_dim;
  if (c.format == NVFP4DA_KV_BF16)
    return make_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, d, rows, d * 2, 64, static_cast<uint32_t>(tile),
                       CU_TENSOR_MAP_SWIZZLE_128B);
  const uint64_t bytes = c.format == NVFP4DA_KV_E4M3 ? d : d / 2;
  return make_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, 128, rows * bytes / 128, 128, 128,
                     static_cast<uint32_t>(tile * bytes / 128), CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace
}  // namespace nvfp4da
