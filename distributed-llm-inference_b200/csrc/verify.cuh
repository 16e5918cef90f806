// Verification of drafted tokens against the target's probabilities (sm_100a).
//
// Sequence b drafted n_b <= T tokens x_i with draft probabilities q_i and has
// target probabilities p_0 .. p_T. Token i is accepted while
// u_i q_i(x_i) < p_i(x_i) (the product rounded to FP32; without draft
// probabilities q_i(x_i) = 1). With a accepted tokens the next one is drawn
// from w = max(p_a - q_a, 0) when x_a was rejected (without draft
// probabilities: p_a with x_a taken out), from p_n when all were accepted.
// The drawing inverts the running sum of W_j = floor(min(w_j, 1) 2^40) at
// floor(u sum W): the W_j are 64-bit integers, so their sums are exact and the
// token does not depend on how the vocabulary is split over threads (at most
// 2^23 entries of 2^40 each stay far below 2^63; a weight below 2^-40 counts
// as none). A row whose w are all zero (p_a = q_a up to rounding) falls back
// to p_a; a row without any weight gives token -1.
//
// One cluster of C CTAs per sequence, no workspace and no atomics. Every warp
// of the cluster owns a contiguous segment of the vocabulary: (1) each warp
// sums its segment, (2) the cluster reads all segment sums through distributed
// shared memory and finds the segment that holds the level, (3) its CTA splits
// that segment over its warps the same way and the warp that holds the level
// scans 32 entries at a time. The row is read once from HBM (twice the chosen
// segment, from L2). Bound by HBM at large batches, by the chain of three
// dependent reads at small ones.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace pdb {

struct VerifyParams {
  const int64_t* draft_tokens;   // [B, T]
  const void* target;            // [B, T + 1, V]
  const void* draft;             // [B, T, V] or NULL
  const float* accept_uniforms;  // [B, T]
  const float* sample_uniforms;  // [B]
  const int32_t* draft_lengths;  // [B] or NULL (all T)
  int64_t* tokens;               // [B, T + 1]
  int32_t* counts;               // [B]
  int64_t V;
  int B, T;
};

constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32, kVerifyMaxCluster = 8;

// One row's weights: w_j = p_j - q_j, or p_j with entry `hit` taken out.
template <typename T>
struct VerifyRow {
  const T* p;
  const T* q;
  int64_t hit;
  __device__ __forceinline__ long long weight(float pj, float qj, int64_t j) const {
    float w = __fsub_rn(pj, qj);  // NaN and negative differences count as none
    if (j == hit) w = 0.f;
    return w > 0.f ? __float2ll_rz(fminf(w, 1.f) * 1099511627776.f) : 0ll;
  }
  __device__ __forceinline__ long long at(int64_t j) const {
    return weight(Elem<T>::to_f(p[j]), q ? Elem<T>::to_f(q[j]) : 0.f, j);
  }
  // Sum over [begin, end), lane-strided, several loads in flight.
  __device__ __forceinline__ long long sum(int64_t begin, int64_t end, int lane) const {
    long long s = 0;
    int64_t j = begin + lane;
    for (; j + 7 * 32 < end; j += 8 * 32) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = Elem<T>::to_f(p[j + 32 * i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = q ? Elem<T>::to_f(q[j + 32 * i]) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += weight(a[i], b[i], j + 32 * i);
    }
    for (; j < end; j += 32) s += at(j);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
};

// The part (of `n` sums) that holds `level`, and the sum of those before it.
__device__ __forceinline__ int verify_part(const long long* sums, int n, long long level,
                                           long long* before) {
  long long run = 0;
  for (int i = 0; i < n; ++i) {
    if (run + sums[i] > level) {
      *before = run;
      return i;
    }
    run += sums[i];
  }
  *before = run;
  return n - 1;
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __shared__ long long sums[kVerifyWarps];
  __shared__ long long all[kVerifyMaxCluster * kVerifyWarps];
  __shared__ int s_accepted, s_n;
  __shared__ int64_t s_hit;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / C;
  grid_dependency_wait();
  launch_dependents();

  if (warp == 0) {
    int n = p.draft_lengths ? __ldg(p.draft_lengths + b) : p.T;
    if (n < 0 || n > p.T) {
      raise_error(0x2u);
      n = n < 0 ? 0 : p.T;
    }
    int accepted = 0;
    int64_t hit = -1;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool ok = i < n;
      int64_t x = -1;
      if (ok) {
        x = p.draft_tokens[(int64_t)b * p.T + i];
        ok = x >= 0 && x < p.V;
        if (!ok) raise_error(0x40u);
      }
      if (ok) {
        const float pt = Elem<T>::to_f(
            static_cast<const T*>(p.target)[((int64_t)b * (p.T + 1) + i) * p.V + x]);
        const float qt =
            p.draft ? Elem<T>::to_f(static_cast<const T*>(p.draft)[((int64_t)b * p.T + i) * p.V + x])
                    : 1.f;
        ok = __fmul_rn(p.accept_uniforms[(int64_t)b * p.T + i], qt) < pt;
      }
      const unsigned bad = __ballot_sync(0xffffffffu, i < n && !ok);
      const int here = bad ? __ffs(bad) - 1 : (n - i0 < 32 ? n - i0 : 32);
      accepted += here;
      if (bad) {
        hit = __shfl_sync(0xffffffffu, x, here);
        break;
      }
    }
    if (lane == 0) {
      s_accepted = accepted;
      s_n = n;
      s_hit = hit;
    }
  }
  __syncthreads();
  const int accepted = s_accepted;
  const bool rejected = accepted < s_n;
  VerifyRow<T> row;
  row.p = static_cast<const T*>(p.target) + ((int64_t)b * (p.T + 1) + accepted) * p.V;
  row.q = rejected && p.draft
              ? static_cast<const T*>(p.draft) + ((int64_t)b * p.T + accepted) * p.V
              : nullptr;
  row.hit = rejected && !p.draft ? s_hit : -1;

  const int parts = C * kVerifyWarps;
  const int64_t seg = (p.V + parts - 1) / parts;
  long long total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    const int64_t lo = (int64_t)(rank * kVerifyWarps + warp) * seg;
    const int64_t hi = lo + seg < p.V ? lo + seg : p.V;
    const long long s = row.sum(lo < p.V ? lo : p.V, hi, lane);
    if (lane == 0) sums[warp] = s;
    cluster.sync();
    if (tid < parts)
      all[tid] = cluster.map_shared_rank(sums, tid / kVerifyWarps)[tid % kVerifyWarps];
    cluster.sync();  // every remote read is done: a CTA may rewrite its sums or end
    total = 0;
    for (int i = 0; i < parts; ++i) total += all[i];
    if (total > 0) break;
    row.q = nullptr;  // no weight left after the difference: the target's own
    row.hit = -1;
  }
  long long level = 0;
  const float u = __ldg(p.sample_uniforms + b);
  if (u > 0.f) level = (long long)((double)total * (double)fminf(u, 1.f));
  if (level > total - 1) level = total - 1;
  if (level < 0) level = 0;
  long long before;
  const int part = total > 0 ? verify_part(all, parts, level, &before) : 0;
  if (part / kVerifyWarps != rank) return;
  int64_t* out = p.tokens + (int64_t)b * (p.T + 1);
  for (int i = tid; i <= p.T; i += kVerifyThreads)
    if (i != accepted) out[i] = i < accepted ? p.draft_tokens[(int64_t)b * p.T + i] : -1;
  if (tid == 0) p.counts[b] = accepted + 1;
  if (total <= 0) {
    if (tid == 0) out[accepted] = -1;
    return;
  }
  level -= before;
  // the segment, split over this CTA's warps
  const int64_t s0 = (int64_t)part * seg, s1 = s0 + seg < p.V ? s0 + seg : p.V;
  const int64_t sub = (s1 - s0 + kVerifyWarps - 1) / kVerifyWarps;
  const int64_t lo = s0 + warp * sub < s1 ? s0 + warp * sub : s1, hi = lo + sub < s1 ? lo + sub : s1;
  const long long s = row.sum(lo, hi, lane);
  __syncthreads();
  if (lane == 0) sums[warp] = s;
  __syncthreads();
  const int w = verify_part(sums, kVerifyWarps, level, &before);
  if (w != warp) return;
  level -= before;
  for (int64_t j0 = lo; j0 < hi; j0 += 32) {
    long long run = j0 + lane < hi ? row.at(j0 + lane) : 0ll;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    const unsigned above = __ballot_sync(0xffffffffu, run > level);
    if (above) {
      if (lane == 0) out[accepted] = j0 + (__ffs(above) - 1);
      return;
    }
    level -= __shfl_sync(0xffffffffu, run, 31);
  }
}

}  // namespace pdb
