// Host-side helpers of the C ABI's translation units: error reporting, cached
// kernel attributes, launches and tensor maps.
#pragma once

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <map>
#include <mutex>
#include <utility>

#include "../../include/nvfp4_decoder_attention.h"

// The message nvfp4da_last_error() returns (capi.cu); not exported.
__attribute__((visibility("hidden"))) void nvfp4da_set_last_error(const char* msg);

namespace nvfp4da {
namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  nvfp4da_set_last_error(buf);
  return code;
}

int cuda_fail(cudaError_t e, const char* what) {
  cudaGetLastError();  // clear a non-sticky launch error so later calls start clean
  return fail(NVFP4DA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

#define NVFP4DA_CHECK_LAUNCH(what)                       \
  do {                                                   \
    cudaError_t e_ = cudaGetLastError();                 \
    if (e_ != cudaSuccess) return cuda_fail(e_, what);   \
  } while (0)

constexpr int kMaxDevices = 64;
constexpr uint32_t kMaxDynSmem = 227 * 1024;

int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}

int sm_count() {
  static int cached[kMaxDevices] = {0};
  const int dev = current_device();
  if (dev < kMaxDevices && cached[dev]) return cached[dev];
  int n = 148;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev < kMaxDevices) cached[dev] = n;
  return n;
}

// Raise the dynamic shared-memory limit of `fn` on the current device once
// (cached per kernel and device; all instantiations of one kernel template
// share a function type, so the key is the function address).
std::mutex g_smem_mutex;
std::map<std::pair<const void*, int>, uint32_t> g_smem_set;

template <typename F>
cudaError_t ensure_smem(F* fn, uint32_t bytes) {
  const void* key = reinterpret_cast<const void*>(fn);
  const int dev = current_device();
  // Each host thread remembers its last answer: a serving loop launches the
  // same kernels with the same sizes on every call.
  struct Hit {
    const void* key = nullptr;
    int dev = -1;
    uint32_t bytes = 0;
  };
  thread_local Hit hits[8];
  for (const Hit& h : hits)
    if (h.key == key && h.dev == dev && h.bytes >= bytes) return cudaSuccess;
  thread_local int next_hit = 0;
  std::lock_guard<std::mutex> lock(g_smem_mutex);
  auto it = g_smem_set.find({key, dev});
  if (it != g_smem_set.end() && it->second >= bytes) return cudaSuccess;
  // Prefer the largest shared-memory carve-out so that several CTAs (of this
  // kernel and of the kernels chained after it) fit on one SM.
  cudaError_t e = cudaFuncSetAttribute(key, cudaFuncAttributePreferredSharedMemoryCarveout,
                                       static_cast<int>(cudaSharedmemCarveoutMaxShared));
  // The opt-in is needed whenever static + dynamic shared memory passes 48 KB,
  // not only when the dynamic part alone does, so always declare it.
  if (e == cudaSuccess && bytes > 0)
    e = cudaFuncSetAttribute(key, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess) {
    g_smem_set[{key, dev}] = bytes;
    hits[next_hit] = {key, dev, bytes};
    next_hit = (next_hit + 1) % 8;
  }
  return e;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                           bool pdl, unsigned cluster_x, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  if (cluster_x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster_x;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl,
                   Args&&... args) {
  return launch_cluster(kernel, grid, block, smem, stream, pdl, 1u, std::forward<Args>(args)...);
}

// Allow cluster sizes above the portable 8 for `fn` on the current device once.
std::map<std::pair<const void*, int>, bool> g_cluster_set;

template <typename F>
cudaError_t ensure_big_clusters(F* fn) {
  const void* key = reinterpret_cast<const void*>(fn);
  const int dev = current_device();
  std::lock_guard<std::mutex> lock(g_smem_mutex);
  if (g_cluster_set.count({key, dev})) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(key, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) g_cluster_set[{key, dev}] = true;
  return e;
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    cudaGetLastError();
  });
  return fn;
}

bool make_map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t inner, uint64_t outer,
                 uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle swizzle) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {row_bytes};
  const cuuint32_t box[2] = {box_inner, box_outer};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace nvfp4da
