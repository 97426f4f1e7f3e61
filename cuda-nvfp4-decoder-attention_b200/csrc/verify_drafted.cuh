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
// FP32 would move by more than a token's probability.  Rejections of drawn
// children add up: r = max(p - c q, 0) with c the sum of their s.  Given children
// need one sum a node: that of p without all of them, to which those that are yet
// to be tried add their own p(x).
//
// A cluster of CTAs takes a sequence.  Every CTA gathers the children's p(x) and
// q(x) first, so that the walk reads shared memory, and walks by itself.  A row is
// cut into segments and these into sixteen runs, each CTA having as many runs as
// another; a warp has all of a segment (16 elements a lane) in flight at once.  The
// CTAs exchange the sums of their runs, and one warp looks for the border of u_0 in
// the segment that holds it.  (Every segment's sum to every CTA: 64 trees over
// 128,000 tokens 51 us for 48.)  Which elements make a sum, and in which order,
// follows from the vocabulary alone: the same bits whatever the number of CTAs,
// which follows from the batch and the GPU.
//
// What bounds it: the sequence with the most rejections, one after another (a sum
// needs the one before it).  64 trees of 8 over 128,000 tokens: 42 to 49 us by the
// numbers drawn, 1.5 sums a sequence and five at most, the first of which read 64 MB
// from HBM; 48 trees of 13 given candidates over 49,999 tokens 17 to 19.5 us, one sum a
// node (one a rejection: 72 us); one chain over 32,000 tokens 8.2 us.  Per element two conversions to FP64 and
// three FP64 operations; elements are checked with an integer maximum a piece, and
// cleaned one by one only where that finds one (all of them cleaned: 68 us for 57).
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace nvfp4da {

constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxNodes = 1024, kVerifyMaxCluster = 16;
constexpr int kVerifyRuns = kVerifyMaxCluster;  // of a row's segments
constexpr int kVerifyPiece = 512;  // elements a warp has in flight
constexpr int kVerifyMaxSegments = 1024;

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
  int pieces, segments;   // of kVerifyPiece elements a segment; segments of a row
  int per_cta;            // segments of a CTA at most
  int64_t* path;          // [B, T]
  int64_t* accepted;      // [B]
  int64_t* next;          // [B]
};

// Shared memory: two sets of the runs' sums, those of the CTA's segments, then of the nodes the sum of p(x) of the
// siblings behind them, p(x), q(x), u, token, parent, path, and the tokens of a node's given children.
constexpr size_t verify_smem(int nodes, int segments) {
  return 2 * kVerifyRuns * 8 + static_cast<size_t>(segments) * 8 + static_cast<size_t>(nodes) * 36;
}

__device__ __forceinline__ double verify_clean(float x) {
  return x > 0.0f && x < INFINITY ? static_cast<double>(x) : 0.0;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_drafted_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  pdl_wait();  // nothing of global memory before this: the launch may overlap the kernel ahead
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  extern __shared__ __align__(16) uint8_t verify_raw[];
  double* s_total = reinterpret_cast<double*>(verify_raw);  // [2][kVerifyRuns]
  double* s_part = s_total + 2 * kVerifyRuns;               // [per_cta]
  double* s_behind = s_part + p.per_cta;
  float* s_p = reinterpret_cast<float*>(s_behind + p.nodes);
  float* s_q = s_p + p.nodes;
  float* s_u = s_q + p.nodes;
  int* s_token = reinterpret_cast<int*>(s_u + p.nodes);  // -1: no child
  int* s_parent = s_token + p.nodes;
  int* s_path = s_parent + p.nodes;
  int* s_given = s_path + p.nodes;
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
  __syncthreads();
  if (!draft) {  // a sibling before has the token: once that is rejected, nothing of p(x) is left
    for (int t = threadIdx.x; t < nodes; t += kVerifyThreads) {
      const int from = s_parent[t], x = s_token[t];
      for (int i = 1; i < t && from >= 0; ++i)
        if (s_parent[i] == from && s_token[i] == x) s_p[t] = 0.0f;
    }
  }
  auto sync = [&] {
    if (ctas == 1) __syncthreads();
    else cluster.sync();
  };
  sync();  // every CTA has begun: its shared memory may be written

  // What is left of a row, element by element: p - c q, or p without the first `given` of s_given.
  struct Left {
    const float* p;
    const float* q;  // nullptr: p alone
    double c;
    int given;
  };
  // Four elements of a row from `at` on, zeros behind its end.
  auto fetch4 = [&](const float* row, int at) {
    if (p.vec && at + 4 <= p.vocab) return __ldg(reinterpret_cast<const float4*>(row + at));
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = at + i < p.vocab ? __ldg(row + at + i) : 0.0f;
    return make_float4(x[0], x[1], x[2], x[3]);
  };
  // What is left of them.
  auto rest4 = [&](const Left& l, int at, float4 x, float4 z, double (&r)[4]) {
    r[0] = verify_clean(x.x), r[1] = verify_clean(x.y), r[2] = verify_clean(x.z), r[3] = verify_clean(x.w);
    if (l.q) {
      r[0] = fmax(fma(-l.c, verify_clean(z.x), r[0]), 0.0);
      r[1] = fmax(fma(-l.c, verify_clean(z.y), r[1]), 0.0);
      r[2] = fmax(fma(-l.c, verify_clean(z.z), r[2]), 0.0);
      r[3] = fmax(fma(-l.c, verify_clean(z.w), r[3]), 0.0);
    }
#pragma unroll 1
    for (int i = 0; i < l.given; ++i) {
      const int e = s_given[i] - at;
      r[0] = e == 0 ? 0.0 : r[0];
      r[1] = e == 1 ? 0.0 : r[1];
      r[2] = e == 2 ? 0.0 : r[2];
      r[3] = e == 3 ? 0.0 : r[3];
    }
  };
  const int runs = kVerifyRuns / ctas, run0 = rank * runs;  // this CTA's
  auto first_of = [&](int run) { return run * p.segments / kVerifyRuns; };
  const int seg0 = first_of(run0), seg1 = first_of(run0 + runs);
  int buf = 0;  // s_total's other half holds the last row's sums
  // Sum of what is left.  All threads of the cluster.
  auto sum_left = [&](const Left& l) -> double {
#pragma unroll 1
    for (int seg = seg0 + warp; seg < seg1; seg += kVerifyWarps) {
      double sum = 0.0;
#pragma unroll 1
      for (int k = 0; k < p.pieces; ++k) {
        const int y = (seg * p.pieces + k) * kVerifyPiece;
        if (y >= p.vocab) break;
        float4 x[4], z[4] = {};
        if (p.vec && y + kVerifyPiece <= p.vocab) {  // no branch between the loads: 53 us for 51
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __ldg(reinterpret_cast<const float4*>(l.p + y + 128 * i + 4 * lane));
          if (l.q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = __ldg(reinterpret_cast<const float4*>(l.q + y + 128 * i + 4 * lane));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = fetch4(l.p, y + 128 * i + 4 * lane);
          if (l.q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = fetch4(l.q, y + 128 * i + 4 * lane);
          }
        }
        // Elements as they should be, no negative ones, infinities or NaN: below the bits of infinity.
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top = max(top, max(max(__float_as_uint(x[i].x), __float_as_uint(x[i].y)),
                             max(__float_as_uint(x[i].z), __float_as_uint(x[i].w))));
          top = max(top, max(max(__float_as_uint(z[i].x), __float_as_uint(z[i].y)),
                             max(__float_as_uint(z[i].z), __float_as_uint(z[i].w))));
        }
        // Given children's tokens, out of the lanes that hold them.
#pragma unroll 1
        for (int j = 0; j < l.given; j += 32) {
          const int of = j + lane < l.given ? s_given[j + lane] - y : -1;
          unsigned votes = __ballot_sync(kFull, static_cast<unsigned>(of) < kVerifyPiece);
          while (votes) {
            const int e = __shfl_sync(kFull, of, __ffs(votes) - 1);
            votes &= votes - 1;
            if ((e >> 2 & 31) == lane) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (e >> 7 == i && (e & 3) == 0) x[i].x = 0.0f;
                if (e >> 7 == i && (e & 3) == 1) x[i].y = 0.0f;
                if (e >> 7 == i && (e & 3) == 2) x[i].z = 0.0f;
                if (e >> 7 == i && (e & 3) == 3) x[i].w = 0.0f;
              }
            }
          }
        }
        if (!__any_sync(kFull, top >= 0x7f800000u)) {
          double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
          auto add = [&](double& to, float pv, float qv) {
            const double r = l.q ? fma(-l.c, static_cast<double>(qv), static_cast<double>(pv)) : static_cast<double>(pv);
            if (r > 0.0) to += r;
          };
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            add(s0, x[i].x, z[i].x);
            add(s1, x[i].y, z[i].y);
            add(s2, x[i].z, z[i].z);
            add(s3, x[i].w, z[i].w);
          }
          sum += (s0 + s1) + (s2 + s3);
        } else {
#pragma unroll 1
          for (int at = y + 4 * lane; at < y + kVerifyPiece; at += 128) {
            double r[4];
            rest4(l, at, fetch4(l.p, at), l.q ? fetch4(l.q, at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f), r);
            sum += (r[0] + r[1]) + (r[2] + r[3]);
          }
        }
      }
      sum = warp_sum_f64(sum);
      if (lane == 0) s_part[seg - seg0] = sum;
    }
    __syncthreads();
    for (int run = run0 + warp; run < run0 + runs; run += kVerifyWarps) {
      double own = 0.0;
      for (int i = first_of(run) + lane; i < first_of(run + 1); i += 32) own += s_part[i - seg0];
      own = warp_sum_f64(own);
      if (lane < ctas) cluster.map_shared_rank(s_total, lane)[buf * kVerifyRuns + run] = own;
    }
    sync();
    const double all = warp_sum_f64(lane < kVerifyRuns ? s_total[buf * kVerifyRuns + lane] : 0.0);
    buf ^= 1;
    return all;
  };

  // ---- the walk: the same in every thread of the cluster
  int node = 0, length = 1;
  bool open = true, summed = false;  // summed: the last sums are those of `left`
  double scale = 1.0, total = 0.0;   // s; sum of `left`
  Left left{target, nullptr, 0.0, 0};
  // The first child of `node` behind node t, `nodes`: none.
  auto child_behind = [&](int t) {
    for (int base = t + 1; base < nodes; base += 32) {
      const unsigned votes = __ballot_sync(kFull, base + lane < nodes && s_parent[base + lane] == node);
      if (votes) return base + __ffs(votes) - 1;
    }
    return nodes;
  };
  for (int t = child_behind(0); t < nodes && open; t = child_behind(t)) {
    const double u = s_u[t], pv = verify_clean(s_p[t]), q = draft ? verify_clean(s_q[t]) : 1.0;
    const bool take = u * q * scale < (left.q ? fmax(fma(-left.c, q, pv), 0.0) : pv);
    if (take) {
      if (threadIdx.x == 0) s_path[length] = t;
      ++length;
      node = t;
      scale = 1.0;
      summed = false;
      left = {target + node * p.target_stride[1], nullptr, 0.0, 0};
      continue;
    }
    if (draft) {
      left.q = draft + node * p.draft_stride[1];
      left.c += scale;
      scale = total = sum_left(left);
      summed = true;
    } else {
      if (!summed) {  // the node's first rejection
        __syncthreads();  // s_given is read
        int n = 0;
        for (int base = t; base < nodes; base += 32) {
          const bool mine = base + lane < nodes && s_parent[base + lane] == node;
          const unsigned votes = __ballot_sync(kFull, mine);
          if (mine && warp == 0) s_given[n + __popc(votes & ((1u << lane) - 1u))] = s_token[base + lane];
          n += __popc(votes);
        }
        left.given = n;
        if (warp == 0) {  // from the last node on; nothing is subtracted, so that the smallest p(x) stay
          double carry = 0.0;
          for (int base = nodes - 1; base >= t; base -= 32) {
            const int i = base - lane;
            double behind = i >= t && i + 1 < nodes && s_parent[i + 1] == node ? verify_clean(s_p[i + 1]) : 0.0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double x = __shfl_up_sync(kFull, behind, o);
              if (lane >= o) behind += x;
            }
            behind += carry;
            if (i >= t) s_behind[i] = behind;
            carry = __shfl_sync(kFull, behind, 31);
          }
        }
        __syncthreads();
        total = sum_left(left);
        summed = true;
      }
      // s: what is left without the children so far, those to come still in it
      scale = total + s_behind[t];
    }
    if (scale == 0.0) {
      open = false;
      summed = false;
      left = {target + node * p.target_stride[1], nullptr, 0.0, 0};
    }
  }
  if (!summed) total = sum_left(left);
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
  // The sums before `own` of the lanes, to which the first one belongs whose end passes the border.
  auto before_of = [&](double own) {
    double upto = __shfl_up_sync(kFull, own, 1);
    if (lane == 0) upto = 0.0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(kFull, upto, o);
      if (lane >= o) upto += u;
    }
    return upto;
  };
  const double run_sum = lane < kVerifyRuns ? s_total[(buf ^ 1) * kVerifyRuns + lane] : 0.0;
  double before = before_of(run_sum);
  unsigned holders = __ballot_sync(kFull, before + run_sum > border && run_sum > 0.0);
  const unsigned filled = __ballot_sync(kFull, run_sum > 0.0);
  bool found = holders != 0;
  const int of = found ? __ffs(holders) - 1 : 31 - __clz(filled);
  if (of < run0 || of >= run0 + runs) return;
  before = __shfl_sync(kFull, before, of);
  const int end = first_of(of + 1) - seg0, per_lane = (first_of(of + 1) - first_of(of) + 31) / 32;
  const int i0 = min(first_of(of) - seg0 + lane * per_lane, end), i1 = min(i0 + per_lane, end);
  double own = 0.0;
  for (int i = i0; i < i1; ++i) own += s_part[i];
  int holder = -1, last = -1;
  double run_up = before + before_of(own);
  for (int i = i0; i < i1; ++i) {
    if (s_part[i] > 0.0) last = i;
    if (found && holder < 0 && s_part[i] > 0.0 && run_up + s_part[i] > border) {
      holder = i;
      before = run_up;
    }
    run_up += s_part[i];
  }
  holders = __ballot_sync(kFull, holder >= 0);
  const unsigned lasts = __ballot_sync(kFull, last >= 0);
  found = holders != 0;
  holder = __shfl_sync(kFull, holder, found ? __ffs(holders) - 1 : 0);
  before = __shfl_sync(kFull, before, found ? __ffs(holders) - 1 : 0);
  last = __shfl_sync(kFull, last, lasts ? 31 - __clz(lasts) : 0);
  const int local = found ? holder : last, seg = seg0 + local;
  if (local % kVerifyWarps != warp) return;
  int best = -1;  // the last element so far that is left
#pragma unroll 1
  for (int y = seg * p.pieces * kVerifyPiece; y < min((seg + 1) * p.pieces * kVerifyPiece, p.vocab); y += 128) {
    const int at = y + 4 * lane;
    double r[4];
    rest4(left, at, fetch4(left.p, at), left.q ? fetch4(left.q, at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f), r);
    const double sum = (r[0] + r[1]) + (r[2] + r[3]);
    double scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(kFull, scan, o);
      if (lane >= o) scan += u;
    }
    int hit = -1, any = -1;
    double run = before + (scan - sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      run += r[e];
      if (r[e] > 0.0) any = at + e;
      if (found && hit < 0 && r[e] > 0.0 && run > border) hit = at + e;
    }
    const unsigned hits = __ballot_sync(kFull, hit >= 0), anys = __ballot_sync(kFull, any >= 0);
    if (hits) {
      best = __shfl_sync(kFull, hit, __ffs(hits) - 1);
      break;
    }
    if (anys) best = __shfl_sync(kFull, any, 31 - __clz(anys));
    before += __shfl_sync(kFull, scan, 31);
  }
  if (lane == 0) p.next[b] = best;
}

}  // namespace nvfp4da
