// Verification of drafted tokens against the target's probabilities, from given
// random numbers.  (No counterpart in the reference, which decodes one token.)
//
// The nodes of sequence b's tree are its drafted tokens, parents first; node 0 is
// the token that the last step ended with and is accepted.  With p = the target's
// row at the node last accepted and q = the draft's row there, its children are
// tried in order, each against what the rejections before it left of p:
//   r = p, s = 1;   child c with token x and random number u_c:
//   accepted where u_c q(x) s < r(x): the walk goes on at c;
//   else r = max(r - s q, 0), s = sum r.
// Children drawn independently from q then follow the target's distribution.  A
// draft without probabilities (a search, the k likeliest tokens) has q = 1 at x:
// a rejection takes x out of r.  Where nothing is left (s = 0) the row p itself
// stands again and no further child is tried.  The next token is the first y with
// sum_{z <= y} r(z) > u_0 sum r.  Elements of p and q that are not positive and
// finite count as 0; a child whose token is outside the vocabulary is none; a row
// without positive elements gives token -1.
//
// All of r, s and the sums are FP64: token numbers are borders of sums, which
// FP32 would move by more than a token's probability.
//
// A cluster of CTAs takes a sequence.  Every CTA gathers the children's p(x) and
// q(x) first, so that the walk reads shared memory, and walks by itself; a sum
// over the vocabulary is cut into one contiguous segment a warp, whose sums all
// CTAs exchange and add in the same order (the same bits everywhere).  The warp
// whose segment holds the border of u_0 looks for it.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace nvfp4da {

constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxNodes = 1024, kVerifyMaxCluster = 16;

struct VerifyParams {
  const float* target;  // [B, T, V] by strides over b and t
  const float* draft;   // the same, or nullptr
  int64_t target_stride[2], draft_stride[2];
  const int64_t* tokens;    // [B, T]
  const int64_t* parents;   // [B, T] by parent_stride (0: one for all), or nullptr: t - 1
  int64_t parent_stride;
  const float* uniforms;  // [B, T]
  const int64_t* counts;  // [B] or nullptr: nodes of the tree
  int nodes, vocab;       // T, V
  int vec;                // rows are 16-byte aligned
  int64_t* path;          // [B, T]
  int64_t* accepted;      // [B]
  int64_t* next;          // [B]
};

// Shared memory of the nodes: p(x), q(x), u, token, parent, path, rejected children; then s of each rejection.
constexpr size_t verify_smem(int nodes) { return static_cast<size_t>(nodes) * 28 + 8 + (nodes + 1) * 8; }

__device__ __forceinline__ double verify_clean(float x) {
  return x > 0.0f && x < INFINITY ? static_cast<double>(x) : 0.0;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_drafted_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  extern __shared__ __align__(16) uint8_t verify_raw[];
  __shared__ double s_part[2][kVerifyMaxCluster * kVerifyWarps];
  double* s_scale = reinterpret_cast<double*>(verify_raw);  // s after each rejection at the node
  float* s_p = reinterpret_cast<float*>(s_scale + p.nodes + 1);
  float* s_q = s_p + p.nodes;
  float* s_u = s_q + p.nodes;
  int* s_token = reinterpret_cast<int*>(s_u + p.nodes);  // -1: no child
  int* s_parent = s_token + p.nodes;
  int* s_path = s_parent + p.nodes;
  int* s_gone = s_path + p.nodes;  // tokens rejected at the node
  const int64_t b = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int nodes = p.nodes;
  if (p.counts) nodes = static_cast<int>(min(max(p.counts[b], int64_t(0)), static_cast<int64_t>(p.nodes)));
  if (nodes == 0) {  // a row of the batch without a tree (the whole cluster)
    if (rank == 0) {
      for (int t = threadIdx.x; t < p.nodes; t += kVerifyThreads) p.path[b * p.nodes + t] = -1;
      if (threadIdx.x == 0) {
        p.accepted[b] = 0;
        p.next[b] = -1;
      }
    }
    return;
  }
  const float* target = p.target + b * p.target_stride[0];
  const float* draft = p.draft ? p.draft + b * p.draft_stride[0] : nullptr;
  for (int t = threadIdx.x; t < nodes; t += kVerifyThreads) {
    const int64_t x = p.tokens[b * p.nodes + t];
    const int64_t from = p.parents ? p.parents[b * p.parent_stride + t] : t - 1;
    const bool child = t > 0 && from >= 0 && from < t && x >= 0 && x < p.vocab;
    s_token[t] = child ? static_cast<int>(x) : -1;
    s_parent[t] = child ? static_cast<int>(from) : -1;
    s_u[t] = p.uniforms[b * p.nodes + t];
    s_p[t] = child ? target[from * p.target_stride[1] + x] : 0.0f;
    s_q[t] = child && draft ? draft[from * p.draft_stride[1] + x] : 1.0f;
  }
  cluster.sync();  // every CTA has begun: its shared memory may be written

  // This warp's segment of a row.
  const int segments = ctas * kVerifyWarps, mine = rank * kVerifyWarps + warp;
  const int seg = static_cast<int>(((static_cast<int64_t>(p.vocab) + segments - 1) / segments + 3) / 4 * 4);
  const int y0 = static_cast<int>(min(static_cast<int64_t>(mine) * seg, static_cast<int64_t>(p.vocab)));
  const int y1 = min(y0 + min(seg, p.vocab - y0), p.vocab);

  // What `level` rejections have left of p at token y.
  auto left = [&](float pv, float qv, int y, int level) -> double {
    double r = verify_clean(pv);
    if (draft) {
      const double q = verify_clean(qv);
      for (int l = 0; l < level; ++l) r = fmax(r - s_scale[l] * q, 0.0);
    } else {
      for (int l = 0; l < level; ++l)
        if (s_gone[l] == y) r = 0.0;
    }
    return r;
  };
  // Four elements of a row from y on, of those below y1.
  auto load4 = [&](const float* row, int y, float (&x)[4]) {
    if (p.vec && y + 4 <= y1) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(row + y));
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = y + i < y1 ? __ldg(row + y + i) : 0.0f;
    }
  };
  int buf = 0;
  // Sum of what is left at `node`, the segments' sums in s_part[buf ^ 1].  All threads of the cluster.
  auto total_left = [&](int node, int level) -> double {
    const float* pr = target + node * p.target_stride[1];
    const float* qr = draft ? draft + node * p.draft_stride[1] : nullptr;
    double sum = 0.0;
    for (int y = y0 + 4 * lane; y < y1; y += 128) {
      float x[4], z[4] = {};
      load4(pr, y, x);
      if (qr && level) load4(qr, y, z);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += left(x[i], z[i], y + i, level);
    }
    sum = warp_sum_f64(sum);
    if (lane < ctas) cluster.map_shared_rank(s_part[buf], lane)[mine] = sum;
    cluster.sync();
    const double* part = s_part[buf];
    buf ^= 1;
    double all = 0.0;
    for (int i = lane; i < segments; i += 32) all += part[i];
    return warp_sum_f64(all);
  };

  // ---- the walk: the same in every thread of the cluster
  int node = 0, length = 1, level = 0;
  double scale = 1.0;
  bool open = true, summed = false;  // summed: s_part[buf ^ 1] holds the present row's sums
  for (int t = 1; t < nodes; ++t) {
    if (s_parent[t] != node || !open) continue;
    const int x = s_token[t];
    const double q = verify_clean(s_q[t]), r = left(s_p[t], s_q[t], x, level);
    if (static_cast<double>(s_u[t]) * q * scale < r) {
      node = t;
      level = 0;
      scale = 1.0;
      summed = false;
      if (threadIdx.x == 0) s_path[length] = t;
      ++length;
      continue;
    }
    __syncthreads();  // the lists are read
    if (threadIdx.x == 0) {
      s_scale[level] = scale;
      s_gone[level] = x;
    }
    __syncthreads();
    scale = total_left(node, ++level);
    summed = true;
    if (scale == 0.0) {
      open = false;
      level = 0;
      summed = false;
    }
  }
  const double total = summed ? scale : total_left(node, 0);
  const double* part = s_part[buf ^ 1];
  __syncthreads();
  if (rank == 0) {
    for (int t = threadIdx.x; t < p.nodes; t += kVerifyThreads)
      p.path[b * p.nodes + t] = t == 0 ? 0 : (t < length ? s_path[t] : -1);
    if (threadIdx.x == 0) {
      p.accepted[b] = length;
      if (total == 0.0) p.next[b] = -1;
    }
  }
  if (total == 0.0) return;

  // ---- the next token: the first segment whose end passes u_0 sum r, else the last with anything in it
  const double border = static_cast<double>(s_u[0]) * total;
  const int per_lane = (segments + 31) / 32, i0 = lane * per_lane, i1 = min(i0 + per_lane, segments);
  double own = 0.0;
  for (int i = i0; i < i1; ++i) own += part[i];
  double upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(kFull, upto, o);
    if (lane >= o) upto += u;
  }
  int holder = -1, last = -1;
  double before = 0.0, run_up = upto - own;
  for (int i = i0; i < i1; ++i) {
    if (part[i] > 0.0) last = i;
    if (holder < 0 && run_up + part[i] > border) {
      holder = i;
      before = run_up;
    }
    run_up += part[i];
  }
  const unsigned holders = __ballot_sync(kFull, holder >= 0), lasts = __ballot_sync(kFull, last >= 0);
  holder = __shfl_sync(kFull, holder, holders ? __ffs(holders) - 1 : 0);
  before = __shfl_sync(kFull, before, holders ? __ffs(holders) - 1 : 0);
  last = __shfl_sync(kFull, last, lasts ? 31 - __clz(lasts) : 0);
  const bool found = holder >= 0;
  if (mine != (found ? holder : last)) return;
  const float* pr = target + node * p.target_stride[1];
  const float* qr = draft ? draft + node * p.draft_stride[1] : nullptr;
  int best = -1;  // the last element so far that is left
  for (int base = y0; base < y1; base += 128) {
    const int y = base + 4 * lane;
    float x[4], z[4] = {};
    double r[4] = {}, sum = 0.0;
    if (y < y1) {
      load4(pr, y, x);
      if (qr && level) load4(qr, y, z);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[i] = left(x[i], z[i], y + i, level);
        sum += r[i];
      }
    }
    double scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(kFull, scan, o);
      if (lane >= o) scan += u;
    }
    int hit = -1, any = -1;
    double run = before + (scan - sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      run += r[i];
      if (r[i] > 0.0) any = y + i;
      if (found && hit < 0 && r[i] > 0.0 && run > border) hit = y + i;
    }
    const unsigned hits = __ballot_sync(kFull, hit >= 0), anys = __ballot_sync(kFull, any >= 0);
    if (anys) best = __shfl_sync(kFull, any, 31 - __clz(anys));
    if (hits) {
      best = __shfl_sync(kFull, hit, __ffs(hits) - 1);
      break;
    }
    before += __shfl_sync(kFull, scan, 31);
  }
  if (lane == 0) p.next[b] = best;
}

}  // namespace nvfp4da
