// C ABI of serving drafted tokens from a paged KV cache: pages reserved and
// given back, rows by slots, attention through the block table, and the
// verification of drafted tokens.
// Declarations: include/nvfp4_decoder_attention.h.
#include <algorithm>
#include <cmath>

#include "host_util.cuh"
#include "kv_host.cuh"
#include "page_table.cuh"
#include "paged_general.cuh"
#include "paged_kv.cuh"
#include "tree_attention.cuh"
#include "tree_launch.cuh"
#include "verify_drafted.cuh"

namespace nvfp4da {
namespace {

int check_table(const nvfp4da_page_table* t, PageTableParams& p) {
  if (!t) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "the page table is NULL");
  if (!t->pages || !t->held || !t->free_pages || !t->free_count)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "a field of the page table is NULL");
  if (t->batch <= 0 || t->max_pages <= 0 || t->pool <= 0 || t->page_size <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "the page table's dimensions must all be positive");
  if (t->page_size % NVFP4DA_PAGE_SIZE_MULTIPLE != 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "the page size must be a multiple of %d, got %lld",
                NVFP4DA_PAGE_SIZE_MULTIPLE, static_cast<long long>(t->page_size));
  if (!product_within(t->batch, t->max_pages, kI32Max) || !product_within(t->max_pages, t->page_size, kI32Max / 2) ||
      !product_within(t->pool, t->page_size, kI32Max))
    return fail(NVFP4DA_ERR_UNSUPPORTED,
                "a page table holds fewer than 2^31 entries, 2^30 positions a sequence and 2^31 slots in its pool");
  p.table = t->pages;
  p.held = t->held;
  p.free_pages = t->free_pages;
  p.free_count = t->free_count;
  p.batch = static_cast<int>(t->batch);
  p.max_pages = static_cast<int>(t->max_pages);
  p.pages = static_cast<int>(t->pool);
  p.page_size = static_cast<int>(t->page_size);
  return NVFP4DA_OK;
}

// Query rows per KV head from which tree_tc_kernel runs.  Streaming / tcgen05, us, 6 KV heads (64 rows: 4), 8 sequences
// of 200 to 400 positions, 32 of 100 to 4,000, 8 of 8,000 to 12,000, pages of 32; head_dim 128:
//          8 rows                   12 rows                  20 rows                  64 rows
//   BF16   23/24   61/62   73/75    24/24   65/62   75/75    28/24   85/62   85/74    40/23  124/52  124/60
//   E4M3   24/30   46/77   52/77    26/30   54/79   60/77    30/30   79/77   88/83    46/30  110/64  120/69
//   NVFP4  24/32   46/77   48/75    26/32   60/79   67/75    32/30   89/73   99/75    46/30  120/61  134/67
// and head_dim 64:
//   BF16   19/22   44/50   48/54    19/22   50/50   50/54    24/22   67/50   65/54    32/22  101/42   91/46
//   E4M3   22/26   36/67   36/63    22/26   44/67   46/64    26/26   60/65   67/67    36/26   83/54   89/56
//   NVFP4  22/26   36/65   38/62    23/26   46/67   50/62    26/26   67/64   75/66    38/26   89/54   97/54
constexpr int64_t paged_tc_min_rows(int64_t head_dim, int format) {
  return format == NVFP4DA_KV_BF16 ? (head_dim == 64 ? 17 : 9) : format == NVFP4DA_KV_E4M3 && head_dim == 64 ? 33 : 17;
}

// Groups of 8 query rows that a warp of the streaming kernel holds.  Wider warps decode codes fewer times, but have less
// of a tile each.  Three groups for 17 to 24 rows and two for 25 to 32 are the fastest where decoding counts; where a
// segment is a few tiles, three cost 2 to 4 us more than one.  us for 1, 2, 3 groups, E4M3, head_dim 64, 8 KV heads:
//                                       12 rows          20 rows          24 rows          32 rows
//   37 sequences of 90 to 6,003         64, 64, 76       94, 90, 80       96, 92, 82       98, 94, 119
//   64 of 2,000 to 3,000                88, 88, 107      133, 125, 111    133, 125, 115    137, 129, 168
//   4 of 30,000 to 32,000               66, 64, 74       98, 92, 78       100, 92, 80      102, 94, 119
//   32 of 10 to 300                     25, 27, 33       31, 29, 35       31, 31, 35       33, 31, 41
//   8 of 50 to 600                      21, 21, 24       23, 23, 25       23, 25, 27       25, 25, 29
// 20 rows of 8 sequences of 8,000 to 12,000 at head_dim 128: 106, 113.
int paged_width(int64_t head_dim, int format, int64_t rows) {
  return head_dim != 64 || format != NVFP4DA_KV_E4M3 || rows <= 16 ? 1 : rows <= 24 ? 3 : 2;
}

// CTAs an SM of paged_attn_general_kernel that the splits of the cache's length are to give.  us for 4, 8, 16: 64
// sequences of 1,024 to 8,191 positions, head_dim 96, BF16 249, 260, 240, E4M3 228, 237, 223; 8 x 26,000 E4M3 180, 162,
// 197; 16 of 3,000 to 5,000, head_dim 192, BF16 135, 119, 148; 16 of 100 to 4,000, head_dim 80, 32 rows of NVFP4 49, 57, 80.
constexpr int64_t kPgenPerSm = 8;

template <int FMT, int KS>
cudaError_t launch_paged_general(dim3 grid, const TreeAttnParams& p, const PagedView& pg, cudaStream_t s) {
  auto* kern = paged_attn_general_kernel<FMT, KS>;
  cudaError_t e = ensure_smem(kern, pgen_smem<KS>());
  return e != cudaSuccess ? e : launch(kern, grid, dim3(kPgenThreads), pgen_smem<KS>(), s, true, p, pg);
}

template <int FMT, int KS = 16>
cudaError_t launch_paged_general_d(int64_t head_dim, dim3 grid, const TreeAttnParams& p, const PagedView& pg,
                                   cudaStream_t s) {
  if (head_dim == 16 * KS) return launch_paged_general<FMT, KS>(grid, p, pg, s);
  if constexpr (KS > 1) return launch_paged_general_d<FMT, KS - 1>(head_dim, grid, p, pg, s);
  return cudaErrorInvalidValue;
}

// Plan of the paged attention.
struct PagedPlan {
  bool stream;  // tree_stream_kernel (or tc: tree_tc_kernel), else paged_attn_general_kernel
  bool tc;
  int wide;  // groups of 8 query rows per warp
  int row_chunks, rows_per_pass, passes, tile, box;
  int splits;  // general kernel
  int64_t split_len;
  size_t bytes;
};

int plan_paged(const nvfp4da_kv_cache* c, int64_t batch, int64_t max_pages, int64_t tokens, int64_t q_heads,
               int64_t max_past, PagedPlan& pl) {
  int r = check_pool(c);
  if (r) return r;
  if (batch <= 0 || max_pages <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "the block table's dimensions must all be positive");
  if (!product_within(batch, c->kv_heads, 65535))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "B*Hkv must be at most 65535");
  if (!product_within(max_pages, c->capacity, kI32Max / 2) || !product_within(batch, max_pages, kI32Max))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "a block table holds fewer than 2^31 entries and 2^30 positions a sequence");
  if (tokens <= 0 || q_heads <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "token and query head counts must be positive");
  if (q_heads % c->kv_heads != 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "number of query heads must be divisible by number of KV heads");
  if (max_past < 0) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "max_past_length must be nonnegative");
  const int64_t capacity = max_pages * c->capacity;
  if (tokens > capacity || max_past > capacity - tokens)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "max_past_length + token count exceeds the block table (%lld + %lld > %lld)",
                static_cast<long long>(max_past), static_cast<long long>(tokens), static_cast<long long>(capacity));
  const int64_t group = q_heads / c->kv_heads;
  if (!product_within(group, tokens, 65535) || !product_within(batch * q_heads, tokens, kI32Max))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "too many query rows: (Hq/Hkv)*T must be at most 65535 and B*T*Hq below 2^31");
  const int64_t visible = max_past + tokens, d = c->head_dim, nq = group * tokens;
  // The streaming kernel: tensor-core tiles for these head dimensions; the pool's
  // 128-byte lines and the prefix of the batch have to fit.
  pl.stream = (d == 64 || d == 128 || d == 256) && batch <= kTsMaxBatch && tensor_map_encoder() != nullptr &&
              product_within(c->batch * c->kv_heads * c->capacity, 2, kI32Max);
  pl.tc = pl.stream && d <= 128 && nq >= paged_tc_min_rows(d, c->format);
  // Places of tiles and their order are 32-bit in the kernels.
  if (!product_within(batch * c->kv_heads * (ceil_div(capacity, kTtKeys) + kTtSegment), ceil_div(nq, 8), kI32Max))
    pl.stream = pl.tc = false;
  if (pl.stream) {
    if (pl.tc) {
      pl.passes = static_cast<int>(ceil_div(nq, 2 * kTtRows));
      pl.rows_per_pass = static_cast<int>(ceil_div(nq, pl.passes));
    } else {
      pl.row_chunks = 1;
      pl.wide = paged_width(d, c->format, nq);
      while (pl.row_chunks < kTsWarps && 8 * pl.wide * pl.row_chunks < nq) pl.row_chunks *= 2;
      pl.rows_per_pass = 8 * pl.wide * pl.row_chunks;
      pl.passes = static_cast<int>(ceil_div(nq, pl.rows_per_pass));
    }
    pl.tile = pl.tc ? kTtKeys : c->format == NVFP4DA_KV_BF16 ? kTsTile<kKvFmtBf16> : kTsTile<kKvFmtE4m3>;
    pl.box = static_cast<int>(std::min<int64_t>(pl.tile, c->capacity & -c->capacity));
    pl.bytes = align_up(static_cast<size_t>(2 * sm_count()) * (pl.rows_per_pass * (d * 4 + 8) + 16), 256);
    return NVFP4DA_OK;
  }
  const int64_t base = batch * c->kv_heads * ceil_div(nq, kPgenRows);
  int64_t splits = std::min(ceil_div(kPgenPerSm * sm_count(), base), ceil_div(visible, 2 * kPgenTile));
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, 1024));
  pl.split_len = ceil_div(ceil_div(visible, splits), kPgenTile) * kPgenTile;
  pl.splits = static_cast<int>(ceil_div(visible, pl.split_len));
  const size_t rows = static_cast<size_t>(batch * tokens * q_heads);
  pl.bytes = align_up(pl.splits > 1 ? rows * pl.splits * (c->head_dim + 2) * 4 : 16, 256);
  return NVFP4DA_OK;
}

__global__ void paged_status_kernel(unsigned* flags, int clear) {
  *flags |= clear ? atomicExch(&g_tree_errors, 0u) : atomicOr(&g_tree_errors, 0u);
}

}  // namespace

cudaError_t paged_attention_flags(unsigned* flags, int clear, cudaStream_t s) {
  paged_status_kernel<<<1, 1, 0, s>>>(flags, clear);
  return cudaGetLastError();
}

}  // namespace nvfp4da

using namespace nvfp4da;

extern "C" {

int nvfp4da_reserve_pages(const nvfp4da_page_table* table, const int64_t* past_lengths, const int64_t* counts,
                          int64_t tokens, int64_t* slots, int64_t* granted, void* stream) {
  PageTableParams p{};
  int r = check_table(table, p);
  if (r) return r;
  if (!past_lengths || !slots || !granted || tokens <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "reserve_pages: invalid arguments");
  if (tokens > 1 << 20 || !product_within(table->batch, tokens, kI32Max))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "reserve_pages: at most 2^20 tokens a sequence and fewer than 2^31 in all");
  p.lengths = past_lengths;
  p.counts = counts;
  p.tokens = static_cast<int>(tokens);
  p.by_tokens = page_divisor(static_cast<uint32_t>(tokens));
  p.by_size = page_divisor(static_cast<uint32_t>(p.page_size));
  p.slots = slots;
  p.granted = granted;
  cudaError_t e = launch_cluster(reserve_pages_kernel, dim3(kPageCtas), dim3(kPageThreads), 0,
                                 static_cast<cudaStream_t>(stream), true, kPageCtas, p);
  return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "reserve_pages launch");
}

int nvfp4da_release_pages(const nvfp4da_page_table* table, const int64_t* lengths, void* stream) {
  PageTableParams p{};
  int r = check_table(table, p);
  if (r) return r;
  if (!lengths) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "release_pages: invalid arguments");
  p.lengths = lengths;
  cudaError_t e = launch(release_pages_kernel, dim3(1), dim3(kPageThreads), 0, static_cast<cudaStream_t>(stream), true, p);
  return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "release_pages launch");
}

int nvfp4da_paged_kv_append(const nvfp4da_kv_cache* c, const uint16_t* new_k, const int64_t* k_strides,
                            const uint16_t* new_v, const int64_t* v_strides, int64_t batch, int64_t tokens,
                            const int64_t* slots, int64_t slot_stride, const int64_t* source, int64_t rows,
                            const int64_t* counts, void* stream) {
  int r = check_pool(c);
  if (r) return r;
  if (!new_k || !new_v || !k_strides || !v_strides || !slots || batch <= 0 || tokens <= 0 || rows <= 0 ||
      slot_stride < rows || (!source && rows != tokens))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "paged_kv_append: invalid arguments");
  if (!product_within(batch, c->kv_heads, 65535))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "B*Hkv must be at most 65535");
  if (tokens > kI32Max - kKvThreads || rows > kI32Max - kKvThreads)
    return fail(NVFP4DA_ERR_UNSUPPORTED, "paged_kv_append: too many tokens");
  PagedAppendParams p{};
  p.k = k_store(*c);
  p.v = v_store(*c);
  p.new_k = new_k;
  p.new_v = new_v;
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = k_strides[i];
    p.v_stride[i] = v_strides[i];
  }
  p.slots = slots;
  p.slot_stride = slot_stride;
  p.source = source;
  p.counts = counts;
  p.rows = static_cast<int>(rows);
  p.tokens = static_cast<int>(tokens);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.head_dim = static_cast<int>(c->head_dim);
  p.pages = static_cast<int>(c->batch);
  p.page_size = static_cast<int>(c->capacity);
  p.lanes = lanes_per_row(c->head_dim, 16);
  p.vec_k = row_vector(new_k, k_strides) == 8;
  p.vec_v = row_vector(new_v, v_strides) == 8;
  const dim3 grid(static_cast<unsigned>(ceil_div(rows, kKvThreads / p.lanes)), static_cast<unsigned>(batch * c->kv_heads));
  auto* kernel = c->format == NVFP4DA_KV_BF16   ? paged_append_kernel<kKvFmtBf16>
                 : c->format == NVFP4DA_KV_E4M3 ? paged_append_kernel<kKvFmtE4m3>
                                                : paged_append_kernel<kKvFmtNvfp4>;
  cudaError_t e = launch(kernel, grid, dim3(kKvThreads), 0, static_cast<cudaStream_t>(stream), true, p);
  return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "paged_kv_append launch");
}

int nvfp4da_paged_kv_read(const nvfp4da_kv_cache* c, const int64_t* slots, int64_t batch, int64_t length,
                          uint16_t* k_out, uint16_t* v_out, void* stream) {
  int r = check_pool(c);
  if (r) return r;
  if (!slots || !k_out || !v_out || batch <= 0 || length <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "paged_kv_read: invalid arguments");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "paged_kv_read outputs must be 16-byte aligned");
  if (!product_within(batch, c->kv_heads, 65535))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "B*Hkv must be at most 65535");
  if (length > kI32Max / 2) return fail(NVFP4DA_ERR_UNSUPPORTED, "paged_kv_read: too many rows");
  PagedReadParams p{};
  p.k = k_store(*c);
  p.v = v_store(*c);
  p.slots = slots;
  p.out_k = k_out;
  p.out_v = v_out;
  p.rows = static_cast<int>(length);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.head_dim = static_cast<int>(c->head_dim);
  p.pages = static_cast<int>(c->batch);
  p.page_size = static_cast<int>(c->capacity);
  p.lanes = lanes_per_row(c->head_dim, 8);
  const dim3 grid(static_cast<unsigned>(ceil_div(length, kKvReadRows * (kKvThreads / p.lanes))),
                  static_cast<unsigned>(batch * c->kv_heads));
  auto* kernel = c->format == NVFP4DA_KV_BF16   ? paged_read_kernel<kKvFmtBf16>
                 : c->format == NVFP4DA_KV_E4M3 ? paged_read_kernel<kKvFmtE4m3>
                                                : paged_read_kernel<kKvFmtNvfp4>;
  cudaError_t e = launch(kernel, grid, dim3(kKvThreads), 0, static_cast<cudaStream_t>(stream), true, p);
  return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "paged_kv_read launch");
}

size_t nvfp4da_paged_attention_workspace_size(const nvfp4da_kv_cache* c, int64_t batch, int64_t max_pages,
                                              int64_t tokens, int64_t q_heads, int64_t max_past_length) {
  PagedPlan pl{};
  return plan_paged(c, batch, max_pages, tokens, q_heads, max_past_length, pl) ? 0 : pl.bytes;
}

int nvfp4da_paged_attention(const uint16_t* q, const nvfp4da_kv_cache* c, const int32_t* block_table, int64_t batch,
                            int64_t max_pages, const uint8_t* tree_mask, int64_t mask_batch_stride, uint16_t* context,
                            int64_t tokens, int64_t q_heads, const int64_t* past_lengths, int64_t max_past_length,
                            const int64_t* counts, void* ws, size_t ws_bytes, void* stream) {
  PagedPlan pl{};
  int r = plan_paged(c, batch, max_pages, tokens, q_heads, max_past_length, pl);
  if (r) return r;
  if (!q || !context || !block_table || !past_lengths)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "paged attention: NULL pointer");
  if (!aligned(q, 16) || !aligned(context, 16))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "attention tensors must be 16-byte aligned");
  const bool needs_ws = pl.stream || pl.splits > 1;
  if (needs_ws && (!ws || ws_bytes < pl.bytes))
    return fail(NVFP4DA_ERR_WORKSPACE, "paged attention workspace too small (%zu < %zu bytes)", ws ? ws_bytes : size_t(0),
                pl.bytes);
  if (needs_ws && !aligned(ws, 16))
    return fail(NVFP4DA_ERR_WORKSPACE, "the paged attention workspace must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PagedView pg = {block_table, static_cast<int>(c->batch), static_cast<int>(max_pages),
                        static_cast<int>(c->capacity), counts};
  if (pl.stream) {
    CUtensorMap tk, tv;
    if (!tree_map(&tk, *c, c->k_codes, pl.box) || !tree_map(&tv, *c, c->v_codes, pl.box))
      return fail(NVFP4DA_ERR_CUDA, "tensor map encoding failed for the paged attention");
    TreeStreamParams t{};
    t.q = q;
    t.k = k_store(*c);
    t.v = v_store(*c);
    t.mask = tree_mask;
    t.mask_stride = mask_batch_stride;
    t.ctx = context;
    t.batch = static_cast<int>(batch);
    t.tokens = static_cast<int>(tokens);
    t.q_heads = static_cast<int>(q_heads);
    t.kv_heads = static_cast<int>(c->kv_heads);
    t.group = static_cast<int>(q_heads / c->kv_heads);
    t.capacity = max_pages * c->capacity;
    t.past_lengths = past_lengths;
    t.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(c->head_dim)));
    t.row_chunks = pl.row_chunks;
    t.rows_per_pass = pl.rows_per_pass;
    t.passes = pl.passes;
    t.grid = sm_count();
    t.part_slots = static_cast<int4*>(ws);
    t.part_o = reinterpret_cast<float*>(t.part_slots + 2 * t.grid);
    t.part_ml = reinterpret_cast<float2*>(t.part_o + static_cast<size_t>(2 * t.grid) * pl.rows_per_pass * c->head_dim);
    t.pg = pg;
    t.seg = pl.tc                               ? kTtSegment
            : c->format == NVFP4DA_KV_BF16 ? kTsSegment<kKvFmtBf16>
                                           : kTsSegment<kKvFmtE4m3> + pl.wide - 1;
    t.loaders = pl.box < pl.tile ? 4 : 2;
    while (2 << t.box_log2 <= pl.box) ++t.box_log2;
    if (pl.tc) {
      const bool split = pl.rows_per_pass > kTtRows;
      cudaError_t e = c->format == NVFP4DA_KV_BF16
                          ? launch_tree_tc_d<kKvFmtBf16, true>(c->head_dim, split, tk, tv, t, s)
                      : c->format == NVFP4DA_KV_E4M3
                          ? launch_tree_tc_d<kKvFmtE4m3, true>(c->head_dim, split, tk, tv, t, s)
                          : launch_tree_tc_d<kKvFmtNvfp4, true>(c->head_dim, split, tk, tv, t, s);
      return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "tensor-core paged attention launch");
    }
    cudaError_t e = c->format == NVFP4DA_KV_BF16
                        ? launch_tree_stream_d<kKvFmtBf16, true>(c->head_dim, pl.wide, tk, tv, t, s)
                    : c->format == NVFP4DA_KV_E4M3
                        ? launch_tree_stream_d<kKvFmtE4m3, true>(c->head_dim, pl.wide, tk, tv, t, s)
                        : launch_tree_stream_d<kKvFmtNvfp4, true>(c->head_dim, pl.wide, tk, tv, t, s);
    return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "streaming paged attention launch");
  }
  TreeAttnParams p{};
  p.q = q;
  p.k = k_store(*c);
  p.v = v_store(*c);
  p.mask = tree_mask;
  p.mask_stride = mask_batch_stride;
  p.ctx = context;
  p.partials = static_cast<float*>(ws);
  p.batch = static_cast<int>(batch);
  p.tokens = static_cast<int>(tokens);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.head_dim = static_cast<int>(c->head_dim);
  p.capacity = max_pages * c->capacity;
  p.past_lengths = past_lengths;
  p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(c->head_dim)));
  p.splits = pl.splits;
  p.split_len = pl.split_len;
  const dim3 grid(static_cast<unsigned>(pl.splits),
                  static_cast<unsigned>(ceil_div(q_heads / c->kv_heads * tokens, kPgenRows)),
                  static_cast<unsigned>(batch * c->kv_heads));
  cudaError_t e = c->format == NVFP4DA_KV_BF16   ? launch_paged_general_d<kKvFmtBf16>(c->head_dim, grid, p, pg, s)
                  : c->format == NVFP4DA_KV_E4M3 ? launch_paged_general_d<kKvFmtE4m3>(c->head_dim, grid, p, pg, s)
                                                 : launch_paged_general_d<kKvFmtNvfp4>(c->head_dim, grid, p, pg, s);
  if (e != cudaSuccess) return cuda_fail(e, "paged attention launch");
  if (pl.splits > 1) {
    const int64_t rows = batch * tokens * q_heads;
    tree_combine_kernel<<<static_cast<unsigned>(ceil_div(rows, 4)), 128, 0, s>>>(p);
    NVFP4DA_CHECK_LAUNCH("paged attention combine launch");
  }
  return NVFP4DA_OK;
}

int nvfp4da_verify_drafted(const float* target, const int64_t* target_strides, const float* draft,
                           const int64_t* draft_strides, const int64_t* tokens, const int64_t* parents,
                           int64_t parent_stride, const float* uniforms, const int64_t* counts, int64_t batch,
                           int64_t nodes, int64_t vocab, int64_t* path, int64_t* accepted, int64_t* next_tokens,
                           void* stream) {
  if (!target || !target_strides || (draft && !draft_strides) || !tokens || !uniforms || !path || !accepted ||
      !next_tokens || batch <= 0 || nodes <= 0 || vocab <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "verify_drafted: invalid arguments");
  if (nodes > kVerifyMaxNodes)
    return fail(NVFP4DA_ERR_UNSUPPORTED, "verify_drafted: at most %d nodes a tree, got %lld", kVerifyMaxNodes,
                static_cast<long long>(nodes));
  if (vocab > (1 << 30) || batch > kI32Max / kVerifyMaxCluster)
    return fail(NVFP4DA_ERR_UNSUPPORTED, "verify_drafted: vocabulary or batch too large");
  VerifyParams p{};
  p.target = target;
  p.draft = draft;
  p.vec = aligned(target, 16) && (!draft || aligned(draft, 16));
  for (int i = 0; i < 2; ++i) {
    p.target_stride[i] = target_strides[i];
    p.draft_stride[i] = draft ? draft_strides[i] : 0;
    p.vec = p.vec && p.target_stride[i] % 4 == 0 && p.draft_stride[i] % 4 == 0;
  }
  p.tokens = tokens;
  p.parents = parents;
  p.parent_stride = parent_stride;
  p.uniforms = uniforms;
  p.counts = counts;
  p.nodes = static_cast<int>(nodes);
  p.vocab = static_cast<int>(vocab);
  p.path = path;
  p.accepted = accepted;
  p.next = next_tokens;
  p.pieces = static_cast<int>(ceil_div(ceil_div(vocab, kVerifyPiece), kVerifyMaxSegments));
  p.segments = static_cast<int>(ceil_div(vocab, static_cast<int64_t>(kVerifyPiece) * p.pieces));
  // CTAs a sequence, a power of two: as many as have a segment for every warp and as fit the GPU four to an SM with the
  // rest of the batch.  Twice as many warps a CTA: 48 given trees 23 -> 25 us, 64 trees over 128,000 tokens 53 -> 57, 256
  // over 32,000 43 -> 53.
  const int64_t most = std::min<int64_t>(4LL * sm_count() / batch, ceil_div(p.segments, kVerifyWarps));
  unsigned ctas = 1;
  while (ctas < kVerifyMaxCluster && 2 * ctas <= most) ctas *= 2;
  p.per_cta = static_cast<int>(ceil_div(p.segments, ctas));
  const size_t smem = verify_smem(p.nodes, p.per_cta);
  cudaError_t e = ensure_smem(verify_drafted_kernel, static_cast<uint32_t>(smem));
  if (e == cudaSuccess && ctas > 8) e = ensure_big_clusters(verify_drafted_kernel);
  if (e == cudaSuccess)
    e = launch_cluster(verify_drafted_kernel, dim3(static_cast<unsigned>(batch) * ctas), dim3(kVerifyThreads), smem,
                       static_cast<cudaStream_t>(stream), true, ctas, p);
  return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "verify_drafted launch");
}

}  // extern "C"
