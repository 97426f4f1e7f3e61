// The paged KV cache: rows written and read by slots.  (No counterpart in the
// reference, whose cache reserves C slots a sequence: src/kv_cache.cu:18-57.)
//
// A pool holds N pages of S slots; a page is laid out like the cache of one
// sequence with C = S: codes [N, Hkv, S, D] (kv_quant.cuh's formats, or BF16),
// row scales [N, Hkv, S], block scales [N, Hkv, S, D/16].  Slot s is row s % S of
// page s / S, in every head.  A block table [B, M] names the pages of each
// sequence in order: position j lies in page table[b, j / S], row j % S; an entry
// that names no page of the pool holds nothing (its positions are not seen).
//
// Both kernels move bytes: a lane holds 16 elements of a row of K and of V when
// appending (quantised as kv_quant.cuh does), 8 when reading, several rows in
// flight a thread.  64 sequences x 6 heads of BF16, a row each written and 512 read:
// 36 us, 5.7 TB/s, 0.86 of a copy with both launches; 4 x 2,043 tokens to NVFP4 and
// back 17.6 us, bound by the instructions of both (BF16 packed one by one: 22.5).
#pragma once

#include "common.cuh"
#include "kv_quant.cuh"

namespace nvfp4da {

// A block table over a pool.
struct PagedView {
  const int32_t* table;  // [B, M]
  int pages, max_pages;  // N, M
  int page_size;         // S
  const int64_t* counts; // device [B] or nullptr: rows t >= counts[b] give zeros, and see nothing
};

// The page that holds position pos of sequence b, -1: none.
__device__ __forceinline__ int paged_page(const PagedView& g, int b, int pos) {
  const int i = pos / g.page_size;
  if (i >= g.max_pages) return -1;
  const int page = __ldg(g.table + static_cast<int64_t>(b) * g.max_pages + i);
  return static_cast<unsigned>(page) < static_cast<unsigned>(g.pages) ? page : -1;
}

// Tokens of sequence b that count, of T.
__device__ __forceinline__ int paged_count(const PagedView& g, int b, int tokens) {
  if (!g.counts) return tokens;
  const int64_t n = g.counts[b];
  return n < 0 ? 0 : (n > tokens ? tokens : static_cast<int>(n));
}

struct PagedAppendParams {
  KvStore k, v;
  const uint16_t* new_k;  // [B, T, Hkv, D] by element strides, last dimension contiguous
  const uint16_t* new_v;
  int64_t k_stride[3], v_stride[3];  // batch, token, head
  const int64_t* slots;              // [B, slot_stride]: the slot of a sequence's i-th row
  int64_t slot_stride;
  const int64_t* source;  // [B, rows] or nullptr: token of the i-th row (else i)
  const int64_t* counts;  // [B] or nullptr: rows i >= counts[b] are not written
  int rows, tokens, kv_heads, head_dim;
  int pages, page_size;
  int lanes;         // lanes per row (power of two >= D / 16)
  int vec_k, vec_v;  // 16-byte loads are aligned
};

struct PagedReadParams {
  KvStore k, v;
  const int64_t* slots;  // [B, L]
  uint16_t* out_k;       // [B, Hkv, L, D]
  uint16_t* out_v;
  int rows, kv_heads, head_dim;
  int pages, page_size;
  int lanes;  // lanes per row (power of two >= D / 8)
};

// Row of head h of a slot in [0, N S) (fewer than 2^31 rows).
__device__ __forceinline__ int64_t paged_row(int64_t slot, int page_size, int kv_heads, int h) {
  const uint32_t s = static_cast<uint32_t>(slot), page = s / static_cast<uint32_t>(page_size);
  return static_cast<int64_t>((page * kv_heads + h) * static_cast<uint32_t>(page_size) + s % static_cast<uint32_t>(page_size));
}

// Grid (rows, B * Hkv).
template <int FMT>
__global__ void __launch_bounds__(kKvThreads) paged_append_kernel(const PagedAppendParams p) {
  pdl_launch_dependents();
  pdl_wait();  // nothing of global memory before this: the launch may overlap the kernel ahead
  const int sub = threadIdx.x & (p.lanes - 1);
  const int i = blockIdx.x * (kKvThreads / p.lanes) + threadIdx.x / p.lanes;
  const int h = blockIdx.y % p.kv_heads, b = blockIdx.y / p.kv_heads;
  bool live = i < p.rows && sub * 16 < p.head_dim;
  if (live && p.counts) live = i < p.counts[b];
  int64_t slot = 0, t = i;
  if (live) {
    slot = p.slots[b * p.slot_stride + i];
    if (p.source) t = p.source[static_cast<int64_t>(b) * p.rows + i];
    live = slot >= 0 && slot < static_cast<int64_t>(p.pages) * p.page_size && t >= 0 && t < p.tokens;
  }
  uint32_t wk[8] = {}, wv[8] = {};
  if (live) {
    kv_load16(p.new_k + b * p.k_stride[0] + t * p.k_stride[1] + h * p.k_stride[2] + sub * 16, p.vec_k, wk);
    kv_load16(p.new_v + b * p.v_stride[0] + t * p.v_stride[1] + h * p.v_stride[2] + sub * 16, p.vec_v, wv);
  }
  const int64_t row = live ? paged_row(slot, p.page_size, p.kv_heads, h) : 0;
  if constexpr (FMT == kKvFmtBf16) {
    if (!live) return;
    auto put = [&](const KvStore& st, const uint32_t (&w)[8]) {
      uint4* to = reinterpret_cast<uint4*>(st.codes + (row * p.head_dim + sub * 16) * 2);
      to[0] = make_uint4(w[0], w[1], w[2], w[3]);
      to[1] = make_uint4(w[4], w[5], w[6], w[7]);
    };
    put(p.k, wk);
    put(p.v, wv);
  } else {
    kv_quantize_row<FMT>(wk, p.lanes, sub, live, p.k, row, p.head_dim);
    kv_quantize_row<FMT>(wv, p.lanes, sub, live, p.v, row, p.head_dim);
  }
}

// Grid (rows, B * Hkv); a thread takes kKvReadRows rows.  Slots outside the pool read as zeros.
template <int FMT>
__global__ void __launch_bounds__(kKvThreads) paged_read_kernel(const PagedReadParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int sub = threadIdx.x & (p.lanes - 1), d0 = sub * 8;
  if (d0 >= p.head_dim) return;
  const int step = kKvThreads / p.lanes, h = blockIdx.y % p.kv_heads;
  const int64_t b = blockIdx.y / p.kv_heads;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * step * kKvReadRows + threadIdx.x / p.lanes;
  int64_t slot[kKvReadRows];
#pragma unroll
  for (int i = 0; i < kKvReadRows; ++i) slot[i] = j0 + i * step < p.rows ? __ldg(p.slots + b * p.rows + j0 + i * step) : -1;
  auto inside = [&](int64_t s) { return s >= 0 && s < static_cast<int64_t>(p.pages) * p.page_size; };
  auto out = [&](int64_t j) { return (static_cast<int64_t>(blockIdx.y) * p.rows + j) * p.head_dim + d0; };
  if constexpr (FMT == kKvFmtBf16) {
    uint4 k[kKvReadRows], v[kKvReadRows];
#pragma unroll
    for (int i = 0; i < kKvReadRows; ++i) {
      k[i] = v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (inside(slot[i])) {
        const int64_t at = (paged_row(slot[i], p.page_size, p.kv_heads, h) * p.head_dim + d0) * 2;
        k[i] = __ldg(reinterpret_cast<const uint4*>(p.k.codes + at));
        v[i] = __ldg(reinterpret_cast<const uint4*>(p.v.codes + at));
      }
    }
#pragma unroll
    for (int i = 0; i < kKvReadRows; ++i) {
      const int64_t j = j0 + i * step;
      if (j >= p.rows) return;
      *reinterpret_cast<uint4*>(p.out_k + out(j)) = k[i];
      *reinterpret_cast<uint4*>(p.out_v + out(j)) = v[i];
    }
  } else {
    KvRaw<FMT> k[kKvReadRows], v[kKvReadRows];
#pragma unroll
    for (int i = 0; i < kKvReadRows; ++i)
      if (inside(slot[i])) {
        const int64_t row = paged_row(slot[i], p.page_size, p.kv_heads, h);
        k[i] = kv_fetch8<FMT>(p.k, row, d0, p.head_dim);
        v[i] = kv_fetch8<FMT>(p.v, row, d0, p.head_dim);
      }
#pragma unroll
    for (int i = 0; i < kKvReadRows; ++i) {
      const int64_t j = j0 + i * step;
      if (j >= p.rows) return;
      float x[8];
      kv_decode8<FMT>(k[i], x);
      *reinterpret_cast<uint4*>(p.out_k + out(j)) = kv_pack8(x);
      kv_decode8<FMT>(v[i], x);
      *reinterpret_cast<uint4*>(p.out_v + out(j)) = kv_pack8(x);
    }
  }
}

}  // namespace nvfp4da
