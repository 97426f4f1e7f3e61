// Block tables and slot maps, built on the device from the sequences' lengths.
// (No counterpart in the reference, whose cache reserves C slots a sequence.)
//
// The table [B, M] names the pages each sequence holds, held[b] of them; the
// pages nobody holds stand in free_pages[0 .. free_count), a stack.
//
// Reserve: sequence b gets room for its tokens P_b .. P_b + n_b - 1,
// n_b = counts[b] (T without them) in [0, T]:
//   need_b = max(0, ceil((P_b + n_b) / S) - held_b), 0 where n_b = 0,
// served where need_b = 0 or the needs up to and including b's fit the free
// stack, in the order of the sequences (so the result depends on no timing);
// the pages come from the top.  slots[b, t] = table[b, j / S] S + j % S for
// position j = P_b + t, -1 for t >= n_b, in a page that is not there, and for
// sequences that are not served (granted[b] = 0, their table as it was).
// Release: sequence b keeps ceil(L_b / S) pages; the others go back, the last
// sequence's last page first: a release undoes the reserve before it.  A page stands
// once in the table: references are not counted, and what a row names goes back.
//
// Reserving is one scan over the batch, which every CTA of a cluster of eight does
// for itself, 1,024 sequences at a time; the CTAs share the writing of the table
// and of the slots.  held and free_count change when the whole cluster has read
// them.  Releasing is one CTA's: most steps give back a page or none a sequence.
//
// Latency bounds both: reserving for eight sequences of one token and releasing
// take 12 to 13 us, two launches; 64 prompts of 2,048 tokens (1 MB of slots, 8,000
// pages) 18 us, where one CTA for the slots took 71 and divisions by the compiler 20.
// Four slots in a row a thread, with one division for them, were no faster.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace nvfp4da {

constexpr int kPageThreads = 1024;
constexpr unsigned kPageCtas = 8;
constexpr int kPageLoads = 4;  // loads of a thread in flight
constexpr int kPageFew = 4;    // pages of a sequence that one thread gives back

// Division of x < 2^31 by a fixed d in [1, 2^31): (x + floor(x m / 2^32)) >> s with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1 (Granlund and Montgomery, 1994).
struct PageDivisor {
  uint32_t d, m, s;
};
inline PageDivisor page_divisor(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__device__ __forceinline__ uint32_t page_quotient(uint32_t x, const PageDivisor& v) {
  return (x + __umulhi(x, v.m)) >> v.s;
}

struct PageTableParams {
  int32_t* table;  // [B, M]
  int64_t* held;   // [B]
  int32_t* free_pages;  // [N]
  int64_t* free_count;  // [1]
  int batch, max_pages, pages, page_size;
  const int64_t* lengths;  // P_b or L_b
  const int64_t* counts;   // reserve: [B] or nullptr
  int tokens;              // reserve
  PageDivisor by_tokens, by_size;
  int64_t* slots;          // [B, T]
  int64_t* granted;        // [B]
};

__device__ __forceinline__ int pages_clamp(int64_t x, int most) {
  return x < 0 ? 0 : (x > most ? most : static_cast<int>(x));
}

// Inclusive scan of x over the block's threads in order; `total`: of all.  All threads; ends with a barrier.
__device__ __forceinline__ int pages_scan(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += u;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kPageThreads / 32; ++w) {
    const int s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  total = all;
  __syncthreads();
  return x + before;
}

__global__ void __launch_bounds__(kPageThreads) reserve_pages_kernel(const PageTableParams p) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  pdl_wait();  // nothing of global memory before this: the launch may overlap the kernel ahead
  const int rank = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  __shared__ int s_scan[kPageThreads / 32];
  __shared__ int s_past[kPageThreads], s_count[kPageThreads], s_held[kPageThreads], s_need[kPageThreads],
      s_first[kPageThreads];  // s_first: of the pages taken so far
  const int free_count = pages_clamp(*p.free_count, p.pages);
  const uint32_t size = p.page_size;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t wanted_before = 0;  // needs of the sequences before this chunk: may pass 2^31
  int taken = 0;              // pages, by thread
  for (int base = 0; base < p.batch; base += kPageThreads) {
    const int b = base + threadIdx.x;
    int n = 0, past = 0, held = 0, need = 0;
    if (b < p.batch) {
      const int64_t room = static_cast<int64_t>(p.max_pages) * size, at = p.lengths[b];
      n = p.counts ? pages_clamp(p.counts[b], p.tokens) : p.tokens;
      if (at < 0 || at > room - n) n = 0;
      past = n > 0 ? static_cast<int>(at) : 0;
      held = pages_clamp(p.held[b], p.max_pages);
      if (n > 0) need = max(0, static_cast<int>((past + n + size - 1) / size) - held);
    }
    int total;
    const int upto = pages_scan(need, s_scan, total);
    const bool served = need == 0 || wanted_before + upto <= free_count;
    if (!served) n = need = 0;
    s_past[threadIdx.x] = past;
    s_count[threadIdx.x] = n;
    s_held[threadIdx.x] = held;
    s_need[threadIdx.x] = need;
    s_first[threadIdx.x] = need ? static_cast<int>(wanted_before) + upto - need : 0;
    taken += need;
    wanted_before += total;
    __syncthreads();
    cluster.sync();  // every CTA has read held of this chunk
    if (rank == 0 && b < p.batch) {
      if (need) p.held[b] = held + need;
      p.granted[b] = n;
    }
    const int chunk = min(kPageThreads, p.batch - base);
    for (int i = rank * (kPageThreads / 32) + warp; i < chunk; i += ctas * (kPageThreads / 32))
      for (int k0 = lane; k0 < s_need[i]; k0 += 32 * kPageLoads) {
        int page[kPageLoads];
#pragma unroll
        for (int u = 0; u < kPageLoads; ++u)
          if (k0 + 32 * u < s_need[i]) page[u] = __ldg(p.free_pages + (free_count - 1 - (s_first[i] + k0 + 32 * u)));
#pragma unroll
        for (int u = 0; u < kPageLoads; ++u)
          if (k0 + 32 * u < s_need[i])
            p.table[static_cast<int64_t>(base + i) * p.max_pages + s_held[i] + k0 + 32 * u] = page[u];
      }
    // Slots: a page number is the old table's, or comes from the stack (the table is being written).
    // Neither is written where it is read here, so that several loads are in flight.
    const uint32_t items = static_cast<uint32_t>(chunk) * p.tokens, step = ctas * kPageThreads;
    for (uint32_t x0 = rank * kPageThreads + threadIdx.x; x0 < items; x0 += kPageLoads * step) {
      int page[kPageLoads], at[kPageLoads];
#pragma unroll
      for (int u = 0; u < kPageLoads; ++u) {
        const uint32_t x = x0 + u * step, i = page_quotient(x, p.by_tokens), t = x - i * p.tokens;
        page[u] = -1;
        if (x < items && static_cast<int>(t) < s_count[i]) {
          const uint32_t j = s_past[i] + t, k = page_quotient(j, p.by_size);
          const int extra = static_cast<int>(k) - s_held[i];
          at[u] = j - k * size;
          page[u] = __ldg(extra < 0 ? p.table + static_cast<int64_t>(base + i) * p.max_pages + k
                                    : p.free_pages + (free_count - 1 - (s_first[i] + extra)));
        }
      }
#pragma unroll
      for (int u = 0; u < kPageLoads; ++u)
        if (x0 + u * step < items)
          p.slots[static_cast<int64_t>(base) * p.tokens + x0 + u * step] =
              static_cast<unsigned>(page[u]) < static_cast<unsigned>(p.pages)
                  ? static_cast<int64_t>(page[u]) * size + at[u] : -1;
    }
    __syncthreads();
  }
  int total;
  pages_scan(taken, s_scan, total);
  cluster.sync();  // every CTA has read free_count
  if (rank == 0 && threadIdx.x == 0) *p.free_count = free_count - total;
}

// One CTA.
__global__ void __launch_bounds__(kPageThreads) release_pages_kernel(const PageTableParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int s_scan[kPageThreads / 32];
  __shared__ int s_keep[kPageThreads], s_held[kPageThreads], s_back[kPageThreads], s_upto[kPageThreads];
  const int free_count = pages_clamp(*p.free_count, p.pages);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Places on the stack are unsigned: a table may name a page in all of its 2^31 entries, and the free ones come on top.
  const unsigned room_on_stack = p.pages;
  unsigned pushed = 0;
  for (int base = (p.batch - 1) / kPageThreads * kPageThreads; base >= 0; base -= kPageThreads) {
    const int chunk = min(kPageThreads, p.batch - base);
    if (static_cast<int>(threadIdx.x) < chunk) {
      const int b = base + threadIdx.x;
      const int64_t len = p.lengths[b], room = static_cast<int64_t>(p.max_pages) * p.page_size;
      const int held = pages_clamp(p.held[b], p.max_pages);
      const int keep = len >= room ? held : min(held, (pages_clamp(len, static_cast<int>(room)) + p.page_size - 1) / p.page_size);
      s_keep[threadIdx.x] = keep;
      s_held[threadIdx.x] = held;
      if (held != keep) p.held[b] = keep;
    }
    __syncthreads();
    auto entry = [&](int i, int k) { return p.table + static_cast<int64_t>(base + i) * p.max_pages + k; };
    auto named = [&](int page) { return static_cast<unsigned>(page) < static_cast<unsigned>(p.pages); };
    // A sequence's own thread where few of its pages go back (most steps: none or one), else a warp.
    const int i_own = threadIdx.x;
    const int few = i_own < chunk && s_held[i_own] - s_keep[i_own] <= kPageFew ? s_held[i_own] - s_keep[i_own] : -1;
    int own[kPageFew];
    if (few >= 0) {  // pages that go back (entries may name none)
      int n = 0;
#pragma unroll
      for (int k = 0; k < kPageFew; ++k) own[k] = k < few ? *entry(i_own, s_keep[i_own] + k) : -1;
#pragma unroll
      for (int k = 0; k < kPageFew; ++k) n += named(own[k]);
      s_back[i_own] = n;
    }
    for (int i = warp; i < chunk; i += kPageThreads / 32) {
      if (s_held[i] - s_keep[i] <= kPageFew) continue;
      int n = 0;
      for (int k = s_keep[i] + lane; k < s_held[i]; k += 32) n += named(*entry(i, k));
      n = __reduce_add_sync(kFull, n);
      if (lane == 0) s_back[i] = n;
    }
    __syncthreads();
    int total;
    const int mine = static_cast<int>(threadIdx.x) < chunk ? s_back[chunk - 1 - threadIdx.x] : 0;
    const int upto = pages_scan(mine, s_scan, total);  // from the last sequence on
    if (static_cast<int>(threadIdx.x) < chunk) s_upto[chunk - 1 - threadIdx.x] = upto;
    __syncthreads();
    if (few > 0) {
      unsigned to = free_count + pushed + s_upto[i_own] - 1;  // of the first page that goes back
#pragma unroll
      for (int k = 0; k < kPageFew; ++k) {
        if (k < few) *entry(i_own, s_keep[i_own] + k) = -1;
        if (named(own[k])) {
          if (to < room_on_stack) p.free_pages[to] = own[k];
          --to;
        }
      }
    }
    for (int i = warp; i < chunk; i += kPageThreads / 32) {
      if (s_held[i] - s_keep[i] <= kPageFew) continue;
      unsigned to = free_count + pushed + s_upto[i] - 1;
      for (int k = s_keep[i] + lane; k - lane < s_held[i]; k += 32) {
        const int page = k < s_held[i] ? *entry(i, k) : -1;
        const bool back = named(page);
        const unsigned votes = __ballot_sync(kFull, back);
        const unsigned at = to - __popc(votes & ((1u << lane) - 1u));
        if (back && at < room_on_stack) p.free_pages[at] = page;
        if (k < s_held[i]) *entry(i, k) = -1;
        to -= __popc(votes);
      }
    }
    pushed += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.free_count = min(free_count + pushed, room_on_stack);
}

}  // namespace nvfp4da
