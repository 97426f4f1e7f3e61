// C ABI of drafted-token verification: rotary positions of q and k, the
// quantised KV cache and the attention of a tree of drafted tokens.
// Declarations: include/nvfp4_decoder_attention.h.
#include <algorithm>
#include <cmath>

#include "host_util.cuh"
#include "kv_host.cuh"
#include "rope_positions.cuh"
#include "tree_attention.cuh"
#include "tree_launch.cuh"

namespace nvfp4da {
namespace {

// ---------------------------------------------------------------- rotary positions
template <int V, bool ADJACENT>
cudaError_t launch_rope(RopeQkParams p, cudaStream_t s) {
  const int pairs = p.rotary_dim / 2;
  const int64_t per_token = static_cast<int64_t>(p.q_heads + p.kv_heads) * (p.head_dim / V);
  // Tokens per block: enough items for every thread to have one, as far as the
  // (cos, sin) table holds them.
  int64_t tpb = std::max<int64_t>(1, kRopeThreads / per_token);
  if (pairs > 0) tpb = std::min<int64_t>(tpb, kRopeMaxPairs / pairs);
  p.tokens_per_block = static_cast<int>(tpb);
  rope_qk_kernel<V, ADJACENT><<<static_cast<unsigned>(ceil_div(static_cast<int64_t>(p.rows), tpb)), kRopeThreads, 0, s>>>(p);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- tree attention
struct TreePlan {
  bool stream;  // tree_stream_kernel (or tc: tree_tc_kernel), else the general kernel
  bool tc;
  int wide;     // NG: 8-row groups of queries per warp
  int row_chunks, rows_per_pass, passes;
  int splits;   // general kernel
  int64_t split_len;
  size_t bytes;
};

__global__ void tree_status_kernel(unsigned* flags, int clear) {
  *flags = clear ? atomicExch(&g_tree_errors, 0u) : atomicOr(&g_tree_errors, 0u);
}

int plan_tree(const nvfp4da_kv_cache* c, int64_t tokens, int64_t q_heads, int64_t max_past, TreePlan& pl) {
  int r = check_cache(c);
  if (r) return r;
  if (tokens <= 0 || q_heads <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "token and query head counts must be positive");
  if (q_heads % c->kv_heads != 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "number of query heads must be divisible by number of KV heads");
  if (max_past < 0) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "past_length must be nonnegative");
  if (tokens > c->capacity || max_past > c->capacity - tokens)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "past_length + drafted token count exceeds cache capacity (%lld + %lld > %lld)",
                static_cast<long long>(max_past), static_cast<long long>(tokens), static_cast<long long>(c->capacity));
  const int64_t group = q_heads / c->kv_heads;
  if (!product_within(group, tokens, 65535) || !product_within(c->batch * q_heads, tokens, kI32Max))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "too many query rows: (Hq/Hkv)*T must be at most 65535 and B*T*Hq below 2^31");
  const int64_t visible = max_past + tokens, nq = group * tokens;
  const int64_t d = c->head_dim;
  // The streaming kernel: tensor-core tiles for these head dimensions; the
  // tile line of 128-byte lines and the prefix of the batch have to fit.
  pl.stream = (d == 64 || d == 128 || d == 256) && c->batch <= kTsMaxBatch && tensor_map_encoder() != nullptr &&
              product_within(c->batch * c->kv_heads * c->capacity, 2, kI32Max);
  pl.tc = pl.stream && d <= 128 && nq >= tc_min_rows(d, c->format == NVFP4DA_KV_BF16);
  // Tiles and their order are 32-bit in the kernels.
  const int64_t most_passes = ceil_div(nq, 8);
  if (!product_within(c->batch * c->kv_heads * ceil_div(c->capacity, kTtKeys), most_passes, kI32Max))
    pl.stream = pl.tc = false;
  if (pl.tc) {
    pl.passes = static_cast<int>(ceil_div(nq, 2 * kTtRows));
    pl.rows_per_pass = static_cast<int>(ceil_div(nq, pl.passes));
    pl.splits = 1;
    pl.split_len = visible;
    pl.bytes = align_up(static_cast<size_t>(2 * sm_count()) * (pl.rows_per_pass * (d * 4 + 8) + 16), 256);
    return NVFP4DA_OK;
  }
  if (pl.stream) {
    pl.wide = nq > 8 && d <= 128 ? 2 : 1;
    pl.row_chunks = 1;
    while (pl.row_chunks < kTsWarps && 8 * pl.wide * pl.row_chunks < nq) pl.row_chunks *= 2;
    pl.rows_per_pass = 8 * pl.wide * pl.row_chunks;
    pl.passes = static_cast<int>(ceil_div(nq, pl.rows_per_pass));
    pl.splits = 1;
    pl.split_len = visible;
    pl.bytes = align_up(static_cast<size_t>(2 * sm_count()) * (pl.rows_per_pass * (d * 4 + 8) + 16), 256);
    return NVFP4DA_OK;
  }
  const int64_t base = c->batch * c->kv_heads * ceil_div(group * tokens, kTreeWarps);
  int64_t splits = std::min(ceil_div(8LL * sm_count(), base), ceil_div(visible, 128));
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, 1024));
  pl.split_len = ceil_div(ceil_div(visible, splits), 32) * 32;
  pl.splits = static_cast<int>(ceil_div(visible, pl.split_len));
  const size_t rows = static_cast<size_t>(c->batch * tokens * q_heads);
  pl.bytes = align_up(pl.splits > 1 ? rows * pl.splits * (c->head_dim + 2) * 4 : 16, 256);
  return NVFP4DA_OK;
}

}  // namespace
}  // namespace nvfp4da

using namespace nvfp4da;

extern "C" {

int nvfp4da_apply_rope_qk(const uint16_t* q, const int64_t* q_strides, uint16_t* q_out, const uint16_t* k,
                          const int64_t* k_strides, uint16_t* k_out, int64_t batch, int64_t tokens, int64_t q_heads,
                          int64_t kv_heads, int64_t head_dim, const int64_t* positions, int64_t position_stride,
                          const float* inv_freq, int64_t rotary_dim, int interleaved, float attention_factor,
                          void* stream) {
  if (!q || !q_out || !q_strides || batch <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads < 0 || head_dim <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "apply_rope_qk: invalid arguments");
  if (kv_heads > 0 && (!k || !k_out || !k_strides))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "apply_rope_qk: NULL k, k_out or k_strides");
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "rotary_dim must be even, at least 2 and at most head_dim, got %lld",
                static_cast<long long>(rotary_dim));
  if (!positions || !inv_freq) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "apply_rope_qk: NULL positions or inv_freq");
  if (!std::isfinite(attention_factor))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "attention_factor must be finite");
  if (rotary_dim / 2 > kRopeMaxPairs)
    return fail(NVFP4DA_ERR_UNSUPPORTED, "rotary_dim must be at most %d", 2 * kRopeMaxPairs);
  if (!product_within(batch, tokens, kI32Max) || !product_within(q_heads + kv_heads, head_dim, kI32Max / kRopeThreads))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "apply_rope_qk: tensors too large for a one-dimensional grid");
  RopeQkParams p{};
  p.q = q;
  p.k = k;
  p.q_out = q_out;
  p.k_out = k_out;
  int v = row_vector(q, q_strides);
  if (kv_heads > 0) v = std::min(v, row_vector(k, k_strides));
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = q_strides[i];
    p.k_stride[i] = kv_heads > 0 ? k_strides[i] : 0;
  }
  while (v > 1 && (!aligned(q_out, 2 * v) || (kv_heads > 0 && !aligned(k_out, 2 * v)) || head_dim % v != 0)) v /= 2;
  const int64_t unit = interleaved ? rotary_dim : rotary_dim / 2;
  while (v > 1 && unit % v != 0) v /= 2;
  p.positions = positions;
  p.pos_stride = position_stride;
  p.inv_freq = inv_freq;
  p.factor = attention_factor;
  p.rows = static_cast<uint32_t>(batch * tokens);
  p.tokens = static_cast<uint32_t>(tokens);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.head_dim = static_cast<int>(head_dim);
  p.rotary_dim = static_cast<int>(rotary_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (interleaved)
    e = v == 8 ? launch_rope<8, true>(p, s) : v == 4 ? launch_rope<4, true>(p, s) : v == 2 ? launch_rope<2, true>(p, s) : launch_rope<1, true>(p, s);
  else
    e = v == 8 ? launch_rope<8, false>(p, s) : v == 4 ? launch_rope<4, false>(p, s) : v == 2 ? launch_rope<2, false>(p, s) : launch_rope<1, false>(p, s);
  if (e != cudaSuccess) return cuda_fail(e, "apply_rope_qk launch");
  return NVFP4DA_OK;
}

int nvfp4da_kv_quant_append(const nvfp4da_kv_cache* c, const uint16_t* new_k, const int64_t* k_strides,
                            const uint16_t* new_v, const int64_t* v_strides, int64_t tokens, int64_t past_length,
                            const int64_t* past_lengths, const int64_t* counts, void* stream) {
  int r = check_cache(c);
  if (r) return r;
  if (c->format == NVFP4DA_KV_BF16)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "kv_quant_append needs a quantised cache (nvfp4da_kv_cache_append takes BF16)");
  if (!new_k || !new_v || !k_strides || !v_strides || tokens <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "kv_quant_append: invalid arguments");
  if (!past_lengths) {
    if (past_length < 0) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "past_length must be nonnegative");
    if (tokens > c->capacity || past_length > c->capacity - tokens)
      return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "past_length + current token count exceeds cache capacity");
  }
  KvAppendParams p{};
  p.lanes = lanes_per_row(c->head_dim, 16);
  if (tokens > kI32Max - kKvThreads) return fail(NVFP4DA_ERR_UNSUPPORTED, "kv_quant_append: too many tokens");
  p.k = k_store(*c);
  p.v = v_store(*c);
  p.new_k = new_k;
  p.new_v = new_v;
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = k_strides[i];
    p.v_stride[i] = v_strides[i];
  }
  p.vec_k = row_vector(new_k, k_strides) == 8;
  p.vec_v = row_vector(new_v, v_strides) == 8;
  p.batch = static_cast<int>(c->batch);
  p.tokens = static_cast<int>(tokens);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.head_dim = static_cast<int>(c->head_dim);
  p.capacity = c->capacity;
  p.past_length = past_length;
  p.past_lengths = past_lengths;
  p.counts = counts;
  const dim3 grid(static_cast<unsigned>(ceil_div(tokens, kKvThreads / p.lanes)),
                  static_cast<unsigned>(c->batch * c->kv_heads));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->format == NVFP4DA_KV_E4M3) kv_quant_append_kernel<kKvFmtE4m3><<<grid, kKvThreads, 0, s>>>(p);
  else kv_quant_append_kernel<kKvFmtNvfp4><<<grid, kKvThreads, 0, s>>>(p);
  NVFP4DA_CHECK_LAUNCH("kv_quant_append launch");
  return NVFP4DA_OK;
}

int nvfp4da_kv_quant_read(const nvfp4da_kv_cache* c, int64_t start, const int64_t* starts, int64_t length,
                          uint16_t* k_out, uint16_t* v_out, void* stream) {
  int r = check_cache(c);
  if (r) return r;
  if (c->format == NVFP4DA_KV_BF16)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "kv_quant_read needs a quantised cache");
  if (!k_out || !v_out || length <= 0) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "kv_quant_read: invalid arguments");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "kv_quant_read outputs must be 16-byte aligned");
  if (!starts && (start < 0 || length > c->capacity || start > c->capacity - length))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "rows [%lld, %lld + %lld) are not inside the cache capacity %lld",
                static_cast<long long>(start), static_cast<long long>(start), static_cast<long long>(length),
                static_cast<long long>(c->capacity));
  KvReadParams p{};
  p.lanes = lanes_per_row(c->head_dim, 8);
  if (ceil_div(length, kKvReadRows * (kKvThreads / p.lanes)) > kI32Max)
    return fail(NVFP4DA_ERR_UNSUPPORTED, "kv_quant_read: too many rows for the grid");
  p.k = k_store(*c);
  p.v = v_store(*c);
  p.out_k = k_out;
  p.out_v = v_out;
  p.batch = static_cast<int>(c->batch);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.head_dim = static_cast<int>(c->head_dim);
  p.capacity = c->capacity;
  p.length = length;
  p.start = start;
  p.starts = starts;
  const dim3 grid(static_cast<unsigned>(ceil_div(length, kKvReadRows * (kKvThreads / p.lanes))),
                  static_cast<unsigned>(c->batch * c->kv_heads));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->format == NVFP4DA_KV_E4M3) kv_quant_read_kernel<kKvFmtE4m3><<<grid, kKvThreads, 0, s>>>(p);
  else kv_quant_read_kernel<kKvFmtNvfp4><<<grid, kKvThreads, 0, s>>>(p);
  NVFP4DA_CHECK_LAUNCH("kv_quant_read launch");
  return NVFP4DA_OK;
}

size_t nvfp4da_tree_attention_workspace_size(const nvfp4da_kv_cache* c, int64_t tokens, int64_t q_heads,
                                             int64_t max_past_length) {
  TreePlan pl;
  return plan_tree(c, tokens, q_heads, max_past_length, pl) ? 0 : pl.bytes;
}

int nvfp4da_tree_attention(const uint16_t* q, const nvfp4da_kv_cache* c, const uint8_t* tree_mask,
                           int64_t mask_batch_stride, uint16_t* context, int64_t tokens, int64_t q_heads,
                           int64_t past_length, const int64_t* past_lengths, int64_t max_past_length, void* ws,
                           size_t ws_bytes, void* stream) {
  if (!past_lengths) max_past_length = past_length;
  TreePlan pl;
  int r = plan_tree(c, tokens, q_heads, max_past_length, pl);
  if (r) return r;
  if (!q || !context) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "tree attention: NULL pointer");
  if (!aligned(q, 16) || !aligned(context, 16))
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "attention tensors must be 16-byte aligned");
  const bool needs_ws = pl.stream || pl.splits > 1;
  if (needs_ws && (!ws || ws_bytes < pl.bytes))
    return fail(NVFP4DA_ERR_WORKSPACE, "tree attention workspace too small (%zu < %zu bytes)", ws ? ws_bytes : size_t(0),
                pl.bytes);
  if (needs_ws && !aligned(ws, 16))
    return fail(NVFP4DA_ERR_WORKSPACE, "the tree attention workspace must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (pl.stream) {
    CUtensorMap tk, tv;
    const int64_t tile = pl.tc ? kTtKeys : (c->format == NVFP4DA_KV_BF16 ? kTsTile<kKvFmtBf16> : kTsTile<kKvFmtE4m3>);
    if (!tree_map(&tk, *c, c->k_codes, tile) || !tree_map(&tv, *c, c->v_codes, tile))
      return fail(NVFP4DA_ERR_CUDA, "tensor map encoding failed for the tree attention");
    TreeStreamParams t{};
    t.q = q;
    t.k = k_store(*c);
    t.v = v_store(*c);
    t.mask = tree_mask;
    t.mask_stride = mask_batch_stride;
    t.ctx = context;
    t.batch = static_cast<int>(c->batch);
    t.tokens = static_cast<int>(tokens);
    t.q_heads = static_cast<int>(q_heads);
    t.kv_heads = static_cast<int>(c->kv_heads);
    t.group = static_cast<int>(q_heads / c->kv_heads);
    t.capacity = c->capacity;
    t.past_length = past_length;
    t.past_lengths = past_lengths;
    t.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(c->head_dim)));
    t.row_chunks = pl.row_chunks;
    t.rows_per_pass = pl.rows_per_pass;
    t.passes = pl.passes;
    t.grid = sm_count();
    t.part_slots = static_cast<int4*>(ws);
    t.part_o = reinterpret_cast<float*>(t.part_slots + 2 * t.grid);
    t.part_ml = reinterpret_cast<float2*>(t.part_o + static_cast<size_t>(2 * t.grid) * pl.rows_per_pass * c->head_dim);
    if (pl.tc) {
      const bool split = pl.rows_per_pass > kTtRows;
      cudaError_t e = c->format == NVFP4DA_KV_BF16   ? launch_tree_tc_d<kKvFmtBf16>(c->head_dim, split, tk, tv, t, s)
                      : c->format == NVFP4DA_KV_E4M3 ? launch_tree_tc_d<kKvFmtE4m3>(c->head_dim, split, tk, tv, t, s)
                                                     : launch_tree_tc_d<kKvFmtNvfp4>(c->head_dim, split, tk, tv, t, s);
      if (e != cudaSuccess) return cuda_fail(e, "tensor-core tree attention launch");
      return NVFP4DA_OK;
    }
    cudaError_t e = c->format == NVFP4DA_KV_BF16 ? launch_tree_stream_d<kKvFmtBf16>(c->head_dim, pl.wide, tk, tv, t, s)
                    : c->format == NVFP4DA_KV_E4M3
                        ? launch_tree_stream_d<kKvFmtE4m3>(c->head_dim, pl.wide, tk, tv, t, s)
                        : launch_tree_stream_d<kKvFmtNvfp4>(c->head_dim, pl.wide, tk, tv, t, s);
    if (e != cudaSuccess) return cuda_fail(e, "streaming tree attention launch");
    return NVFP4DA_OK;
  }
  TreeAttnParams p{};
  p.q = q;
  p.k = k_store(*c);
  p.v = v_store(*c);
  p.mask = tree_mask;
  p.mask_stride = mask_batch_stride;
  p.ctx = context;
  p.partials = static_cast<float*>(ws);
  p.batch = static_cast<int>(c->batch);
  p.tokens = static_cast<int>(tokens);
  p.q_heads = static_cast<int>(q_heads);
  p.kv_heads = static_cast<int>(c->kv_heads);
  p.head_dim = static_cast<int>(c->head_dim);
  p.capacity = c->capacity;
  p.past_length = past_length;
  p.past_lengths = past_lengths;
  p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(c->head_dim)));
  p.splits = pl.splits;
  p.split_len = pl.split_len;
  p.lanes = std::max(2, lanes_per_row(c->head_dim, 8));
  const int64_t group = q_heads / c->kv_heads;
  const dim3 grid(static_cast<unsigned>(pl.splits), static_cast<unsigned>(ceil_div(group * tokens, kTreeWarps)),
                  static_cast<unsigned>(c->batch * c->kv_heads));
  switch (c->format) {
    case NVFP4DA_KV_BF16: tree_attn_general_kernel<kKvFmtBf16><<<grid, kTreeWarps * 32, 0, s>>>(p); break;
    case NVFP4DA_KV_E4M3: tree_attn_general_kernel<kKvFmtE4m3><<<grid, kTreeWarps * 32, 0, s>>>(p); break;
    default: tree_attn_general_kernel<kKvFmtNvfp4><<<grid, kTreeWarps * 32, 0, s>>>(p); break;
  }
  NVFP4DA_CHECK_LAUNCH("tree attention launch");
  if (pl.splits > 1) {
    const int64_t rows = c->batch * tokens * q_heads;
    tree_combine_kernel<<<static_cast<unsigned>(ceil_div(rows, 4)), 128, 0, s>>>(p);
    NVFP4DA_CHECK_LAUNCH("tree attention combine launch");
  }
  return NVFP4DA_OK;
}

int nvfp4da_tree_attention_sync_status(void* stream, unsigned* flags, int clear) {
  if (!flags) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "flags is NULL");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Read and cleared in one operation: a flag that a kernel on another stream sets meanwhile is kept for the next call.
  unsigned* word = nullptr;
  cudaError_t e = cudaMallocAsync(reinterpret_cast<void**>(&word), sizeof(unsigned), s);
  if (e != cudaSuccess) return cuda_fail(e, "tree attention status read");
  tree_status_kernel<<<1, 1, 0, s>>>(word, clear);
  e = cudaGetLastError();
  if (e == cudaSuccess) e = paged_attention_flags(word, clear, s);
  if (e == cudaSuccess) e = cudaMemcpyAsync(flags, word, sizeof(unsigned), cudaMemcpyDeviceToHost, s);
  const cudaError_t freed = cudaFreeAsync(word, s);
  if (e == cudaSuccess) e = freed;
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  return e == cudaSuccess ? NVFP4DA_OK : cuda_fail(e, "tree attention status read");
}

}  // extern "C"
