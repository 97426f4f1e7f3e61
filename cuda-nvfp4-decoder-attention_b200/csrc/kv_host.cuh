// Host-side checks and views of KV caches, shared by the translation units that
// launch over them.
#pragma once

#include <algorithm>
#include <limits>

#include "host_util.cuh"
#include "kv_quant.cuh"

namespace nvfp4da {
namespace {

constexpr int64_t kI32Max = std::numeric_limits<int32_t>::max();

// a * b <= limit for nonnegative a, b without overflow.
bool product_within(int64_t a, int64_t b, int64_t limit) { return a == 0 || b <= limit / a; }

// Lanes (a power of two) that hold a row `elements` a lane.
int lanes_per_row(int64_t head_dim, int elements) {
  int lanes = 1;
  while (lanes * elements < head_dim) lanes *= 2;
  return lanes;
}

// Elements per access that a strided BF16 tensor's rows allow.
int row_vector(const void* base, const int64_t* strides) {
  int v = 8;
  for (int i = 0; i < 3; ++i)
    while (v > 1 && strides[i] % v != 0) v /= 2;
  while (v > 1 && !aligned(base, 2 * v)) v /= 2;
  return v;
}

// What the caches of sequences and pools of pages have in common.
int check_cache_fields(const nvfp4da_kv_cache* c) {
  if (!c) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (c->format != NVFP4DA_KV_BF16 && c->format != NVFP4DA_KV_E4M3 && c->format != NVFP4DA_KV_NVFP4)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "unknown cache format %d", c->format);
  if (c->batch <= 0 || c->kv_heads <= 0 || c->capacity <= 0 || c->head_dim <= 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "cache dimensions must all be positive");
  if (c->head_dim % 16 != 0 || c->head_dim > 256)
    return fail(NVFP4DA_ERR_UNSUPPORTED, "head_dim must be a multiple of 16 and at most 256, got %lld",
                static_cast<long long>(c->head_dim));
  return NVFP4DA_OK;
}

int check_cache_rows(const nvfp4da_kv_cache* c) {
  if (!product_within(c->batch, c->kv_heads, kI32Max) ||
      !product_within(c->batch * c->kv_heads, c->capacity, kI32Max))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "the cache must have at most 2^31 - 1 rows");
  const void* fields[6] = {c->k_codes, c->v_codes, c->k_row_scales, c->v_row_scales, c->k_block_scales,
                           c->v_block_scales};
  const int used = c->format == NVFP4DA_KV_BF16 ? 2 : (c->format == NVFP4DA_KV_E4M3 ? 4 : 6);
  for (int i = 0; i < used; ++i) {
    if (!fields[i]) return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "a field of the cache is NULL");
    if (!aligned(fields[i], 16))
      return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "every field of the cache must be 16-byte aligned");
  }
  return NVFP4DA_OK;
}

// A cache of B sequences.
int check_cache(const nvfp4da_kv_cache* c) {
  int r = check_cache_fields(c);
  if (r) return r;
  if (!product_within(c->batch, c->kv_heads, 65535))
    return fail(NVFP4DA_ERR_UNSUPPORTED, "B*Hkv must be at most 65535");
  if ((r = check_cache_rows(c))) return r;
  if (c->format != NVFP4DA_KV_BF16 && c->capacity % NVFP4DA_KV_CAPACITY_MULTIPLE != 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "a quantised cache's capacity must be a multiple of %d, got %lld",
                NVFP4DA_KV_CAPACITY_MULTIPLE, static_cast<long long>(c->capacity));
  return NVFP4DA_OK;
}

// A pool of pages: `batch` pages of `capacity` slots.
int check_pool(const nvfp4da_kv_cache* c) {
  int r = check_cache_fields(c);
  if (r) return r;
  if (c->capacity % NVFP4DA_PAGE_SIZE_MULTIPLE != 0)
    return fail(NVFP4DA_ERR_INVALID_ARGUMENT, "the page size must be a multiple of %d, got %lld",
                NVFP4DA_PAGE_SIZE_MULTIPLE, static_cast<long long>(c->capacity));
  return check_cache_rows(c);
}

KvStore k_store(const nvfp4da_kv_cache& c) {
  return {static_cast<uint8_t*>(c.k_codes), c.k_block_scales, c.k_row_scales};
}
KvStore v_store(const nvfp4da_kv_cache& c) {
  return {static_cast<uint8_t*>(c.v_codes), c.v_block_scales, c.v_row_scales};
}

}  // namespace
}  // namespace nvfp4da
