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
// token does not depend on how the vocabulary is split over threads (the at most
// 2^22 entries of 2^40 each stay below 2^63; a weight below 2^-40 counts
// as none). A row whose w are all zero (p_a = q_a up to rounding) falls back
// to p_a; a row without any weight gives token -1.
//
// One cluster of C CTAs per sequence, no workspace and no atomics. Each CTA owns
// a contiguous range of the vocabulary, cut into blocks of 256 K entries that its
// warps take in turn, so that a CTA reads adjacent memory at any time: (1) every
// block's sum goes to shared memory, the CTA's total to every CTA of the cluster
// through distributed shared memory, (2) the totals give the CTA that holds the
// level, its block sums the block, and one warp scans that block. The row is read
// once from HBM (one block twice, from L2). Bound by HBM at large batches, by the
// chain of dependent reads (draft, its probabilities, the row, the block) at small
// ones.
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

constexpr int kVerifyThreads = 256, kVerifyMaxCluster = 8;
constexpr int kVerifyBlocks = 512;  // block sums that a CTA keeps

// One row's weights: w_j = p_j - q_j, or p_j with entry `hit` taken out.
template <typename T>
struct VerifyRow {
  const T* p;
  const T* q;
  int hit;
  bool wide;  // both rows 16-byte aligned
  // The weight in units of 2^-40, in two parts of 20 bits: w = saturate(p - q) (NaN
  // to 0), h = floor(w 2^20), l = floor((w 2^20 - h) 2^20), each read from the
  // mantissa of a sum with 2^23 that is rounded down. Seven instructions; a conversion
  // to a 64-bit integer with its clamps and sums takes more than twice that and
  // bounds the kernel by issue (256 rows of 100003: 43 us).
  static constexpr uint32_t kBias = 0x4B000000u;  // bits of 2^23
  static __device__ __forceinline__ void add(float w, uint32_t& h, uint32_t& l) {
    const float t = __fmaf_rd(w, 1048576.f, 8388608.f);
    const float r = __fmaf_rn(w, 1048576.f, -__fsub_rn(t, 8388608.f));  // exact
    h += __float_as_uint(t);
    l += __float_as_uint(__fmaf_rd(r, 1048576.f, 8388608.f));
  }
  __device__ __forceinline__ long long at(int j) const {
    uint32_t h = 0, l = 0;
    add(__saturatef(__fsub_rn(Elem<T>::to_f(p[j]), q ? Elem<T>::to_f(q[j]) : 0.f)), h, l);
    return j == hit ? 0ll : ((long long)(h - kBias) << 20) + (l - kBias);
  }
  // Sum over the 256 entries from j0 by one warp (those below V), every lane's.
  __device__ __forceinline__ long long sum256(int j0, int V, int lane) const {
    float a[8];
    if (j0 + 256 <= V) {
      if (wide) {
        constexpr int N = Chunk<T>::N, U = 8 / N;
        uint4 x[U], y[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
          x[i] = __ldg(reinterpret_cast<const uint4*>(p + j0) + i * 32 + lane);
        if (q) {
#pragma unroll
          for (int i = 0; i < U; ++i)
            y[i] = __ldg(reinterpret_cast<const uint4*>(q + j0) + i * 32 + lane);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) Chunk<T>::to_f(x[i], a + i * N);
        if (q) {
          float b[8];
#pragma unroll
          for (int i = 0; i < U; ++i) Chunk<T>::to_f(y[i], b + i * N);
#pragma unroll
          for (int i = 0; i < 8; ++i) a[i] = __fsub_rn(a[i], b[i]);
        }
      } else {
        const T* pr = p + j0 + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = Elem<T>::to_f(__ldg(pr + 32 * i));
        if (q) {
          const T* qr = q + j0 + lane;
          float b[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) b[i] = Elem<T>::to_f(__ldg(qr + 32 * i));
#pragma unroll
          for (int i = 0; i < 8; ++i) a[i] = __fsub_rn(a[i], b[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + lane + 32 * i;
        a[i] = 0.f;
        if (j < V) a[i] = __fsub_rn(Elem<T>::to_f(p[j]), q ? Elem<T>::to_f(q[j]) : 0.f);
      }
    }
    uint32_t h = 0, l = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) add(__saturatef(a[i]), h, l);
    // 256 parts of at most 2^20 each: the 32-bit sums wrap only by the biases
    h = __reduce_add_sync(0xffffffffu, h - 8 * kBias);
    l = __reduce_add_sync(0xffffffffu, l - 8 * kBias);
    long long s = ((long long)h << 20) + l;
    if ((unsigned)(hit - j0) < 256u) {  // the entry that is taken out (without q)
      h = l = 0;
      add(__saturatef(Elem<T>::to_f(p[hit])), h, l);
      s -= ((long long)(h - kBias) << 20) + (l - kBias);
    }
    return s;
  }
};

__device__ __forceinline__ long long warp_scan(long long x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// By one warp: the first of `n` <= 32 PER sums whose running sum is above
// `level` (some sum is), and the running sum before it. PER: sums per lane.
template <int PER>
__device__ __forceinline__ int verify_part(const long long* sums, int n, long long level, int lane,
                                           long long* before) {
  long long v[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = lane * PER + i < n ? sums[lane * PER + i] : 0ll;
    mine += v[i];
  }
  long long run = warp_scan(mine, lane);
  const int f = __ffs(__ballot_sync(0xffffffffu, run > level)) - 1;
  run -= mine;  // before this lane's
  int at = 0;
#pragma unroll
  for (int i = 0; i + 1 < PER; ++i)
    if (at == i && run + v[i] <= level) {
      run += v[i];
      ++at;
    }
  *before = __shfl_sync(0xffffffffu, run, f);
  return f * PER + __shfl_sync(0xffffffffu, at, f);
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 4) verify_kernel(const VerifyParams p) {
  constexpr int NT = kVerifyThreads, kWarps = NT / 32;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __shared__ long long totals[2][kVerifyMaxCluster];
  __shared__ long long sums[kVerifyBlocks];
  __shared__ int s_accepted, s_n, s_hit;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / C, V = (int)p.V;
  // every CTA of the cluster runs before any of them writes into another
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  grid_dependency_wait();
  launch_dependents();

  if (warp == 0) {
    int n = p.draft_lengths ? __ldg(p.draft_lengths + b) : p.T;
    int accepted = 0, hit = -1;
    for (int i0 = 0; i0 < p.T; i0 += 32) {
      // drafts past n are read too (and not used), so that no read waits for n
      const int i = i0 + lane;
      const bool in = i < p.T;
      float u = 0.f, pt = 0.f, qt = 1.f;
      int64_t x = -1;
      if (in) {
        u = p.accept_uniforms[(int64_t)b * p.T + i];
        x = p.draft_tokens[(int64_t)b * p.T + i];
      }
      const bool known = x >= 0 && x < V;
      if (known) {
        pt = Elem<T>::to_f(static_cast<const T*>(p.target)[((int64_t)b * (p.T + 1) + i) * V + x]);
        if (p.draft)
          qt = Elem<T>::to_f(static_cast<const T*>(p.draft)[((int64_t)b * p.T + i) * V + x]);
      }
      if (i0 == 0 && (n < 0 || n > p.T)) {
        raise_error(0x2u);
        n = n < 0 ? 0 : p.T;
      }
      const unsigned bad =
          __ballot_sync(0xffffffffu, i < n && !(known && __fmul_rn(u, qt) < pt));
      const int left = n - i0 < 0 ? 0 : n - i0 < 32 ? n - i0 : 32;
      const int here = bad ? __ffs(bad) - 1 : left;
      if (i < n && lane <= here && !known) raise_error(0x40u);
      accepted += here;
      if (bad) hit = __shfl_sync(0xffffffffu, known ? (int)x : -1, here);
      if (bad || left < 32) break;
    }
    if (lane == 0) {
      s_accepted = accepted;
      s_n = n;
      s_hit = hit;
    }
  }
  const float u = __ldg(p.sample_uniforms + b);
  __syncthreads();
  const int accepted = s_accepted;
  const bool rejected = accepted < s_n;
  VerifyRow<T> row;
  row.p = static_cast<const T*>(p.target) + ((int64_t)b * (p.T + 1) + accepted) * V;
  row.q = rejected && p.draft
              ? static_cast<const T*>(p.draft) + ((int64_t)b * p.T + accepted) * V
              : nullptr;
  row.hit = rejected && !p.draft ? s_hit : -1;
  row.wide = ((reinterpret_cast<uintptr_t>(row.p) | reinterpret_cast<uintptr_t>(row.q)) & 15u) == 0;

  // this CTA's range: `blocks` blocks of `size` entries
  const int share = (V + C - 1) / C;
  const int size = 256 * ((share + 256 * kVerifyBlocks - 1) / (256 * kVerifyBlocks));
  const int blocks = (share + size - 1) / size, first = rank * blocks * size;
  constexpr int PER = kVerifyBlocks / 32;
  long long total = 0, before = 0;
  int pass = 0;
  for (;; ++pass) {
#pragma unroll 2
    for (int x = warp; x < blocks; x += kWarps) {
      long long s = 0;
      for (int j = first + x * size; j < first + (x + 1) * size && j < V; j += 256)
        s += row.sum256(j, V, lane);
      if (lane == 0) sums[x] = s;
    }
    __syncthreads();
    if (warp == 0) {
      long long mine = 0;
      for (int i = lane; i < blocks; i += 32) mine += sums[i];
#pragma unroll
      for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      if (C == 1) {
        if (lane == 0) totals[pass][0] = mine;
      }
      if (C > 1) {
        if (pass == 0) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        if (lane < C) cluster.map_shared_rank(&totals[pass][0], lane)[rank] = mine;
      }
    } else if (C > 1 && pass == 0) {
      asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    }
    if (C == 1) __syncthreads();
    else cluster.sync();
    total = before = 0;
    for (int i = 0; i < C; ++i) {
      if (i < rank) before += totals[pass][i];
      total += totals[pass][i];
    }
    if (total > 0 || pass == 1) break;
    row.q = nullptr;  // no weight left after the difference: the target's own
    row.hit = -1;
    row.wide = (reinterpret_cast<uintptr_t>(row.p) & 15u) == 0;
  }
  long long level = 0;
  if (u > 0.f) level = (long long)((double)total * (double)fminf(u, 1.f));
  if (level > total - 1) level = total - 1;
  if (level < 0) level = 0;
  // the CTA that holds the level (without any weight: the first)
  if (total > 0 ? (level < before || level >= before + totals[pass][rank]) : rank != 0) return;
  int64_t* out = p.tokens + (int64_t)b * (p.T + 1);
  if (warp != 0) {
    for (int i = tid - 32; i <= p.T; i += NT - 32)
      if (i != accepted) out[i] = i < accepted ? p.draft_tokens[(int64_t)b * p.T + i] : -1;
    if (tid == 32) p.counts[b] = accepted + 1;
    return;
  }
  if (total <= 0) {
    if (lane == 0) out[accepted] = -1;
    return;
  }
  level -= before;
  const int x = verify_part<PER>(sums, blocks, level, lane, &before);
  level -= before;
  const int lo = first + x * size, hi = lo + size < V ? lo + size : V;
  for (int j0 = lo; j0 < hi; j0 += 256) {
    long long w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = j0 + 32 * i + lane < hi ? row.at(j0 + 32 * i + lane) : 0ll;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long r = warp_scan(w[i], lane);
      const unsigned above = __ballot_sync(0xffffffffu, r > level);
      if (above) {
        if (lane == 0) out[accepted] = j0 + 32 * i + (__ffs(above) - 1);
        return;
      }
      level -= __shfl_sync(0xffffffffu, r, 31);
    }
  }
}

}  // namespace pdb
