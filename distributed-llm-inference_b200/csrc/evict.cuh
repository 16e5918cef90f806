// Eviction from a paged cache by accumulated attention weight (sm_100a).
//
// Per (sequence, kv head) with n cached tokens, m = min(n, budget) stay: the
// last r = min(recent, m) tokens and, of the n - r others, the m - r of
// highest score (NaN lowest, equal scores by lowest index). They keep their
// order and go, K, V and score, to cells 0 .. m - 1 of new pages; every kv head
// keeps its own tokens, as a page holds each head's row separately.
//
// evict_select_kernel: one CTA per (sequence, kv head). Scores become 32-bit
// keys in the order of the floats; the threshold (the largest key that at
// least m - r candidates reach) is found bit by bit from the top, counting the
// candidates at or above a trial key: 32 counts over keys that stay in
// registers, instead of histograms whose few busy bins serialise. Two block
// scans then number the ties and the kept tokens in index order.
// evict_move_kernel: copies rows in 16-byte pieces; bound by HBM.
#pragma once

#include "common.cuh"

namespace pdb {

struct EvictParams {
  void* k_pool;               // [N, bs, KVH, D]
  void* v_pool;
  const float* scores;        // [B, KVH, S]
  const int32_t* tables;      // [B, W]
  const int32_t* lengths;     // [B]
  const int32_t* new_tables;  // [B, W2]
  int32_t* kept;              // [B, KVH, budget]
  int32_t* new_lengths;       // [B]
  float* new_scores;          // [B, KVH, S]
  int64_t num_blocks, S;
  int B, KVH, W, W2, block_size, bs_shift, budget, recent;
  int row_pieces;             // pieces of a row of one head
};

// Sequence b's length, clamped to what the tables and the scores hold.
__device__ __forceinline__ int evict_length(const EvictParams& p, int b) {
  int n = __ldg(p.lengths + b);
  const int64_t table = (int64_t)p.W * p.block_size;
  const int64_t most = table < p.S ? table : p.S;
  if (n < 0 || n > most) {
    raise_error(0x2u);
    n = n < 0 ? 0 : (int)most;
  }
  return n;
}

// Order-preserving key of a score: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t evict_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;

// Sum of `v` over the CTA (every thread gets it); `red` has 2 * kEvictWarps
// words, used alternately so that one barrier per sum is enough.
__device__ __forceinline__ int evict_block_sum(int v, int* red, int& turn) {
  v = __reduce_add_sync(0xffffffffu, v);
  int* r = red + turn * kEvictWarps;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = r[threadIdx.x & (kEvictWarps - 1)];
  // 16 words, each held by two lanes of the warp
  return __reduce_add_sync(0xffffffffu, s) >> 1;
}
// Exclusive prefix of `v` over the CTA's threads, and the CTA's sum.
__device__ __forceinline__ int evict_block_scan(int v, int* red, int& turn, int* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  int* r = red + turn * kEvictWarps;
  turn ^= 1;
  if (lane == 31) r[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kEvictWarps; ++w) {
    if (w < warp) before += r[w];
    all += r[w];
  }
  *sum = all;
  return before + inc - v;
}

// Candidates per round of the CTA: E consecutive ones per thread.
template <int E>
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int red[2 * kEvictWarps];
  int turn = 0;
  const int bh = blockIdx.x, b = bh / p.KVH, tid = threadIdx.x;
  grid_dependency_wait();
  launch_dependents();
  const int n = evict_length(p, b);
  const int m = n < p.budget ? n : p.budget;
  const int r = p.recent < m ? p.recent : m;
  const int cand = n - r, want = m - r;
  const float* sc = p.scores + (int64_t)bh * p.S;
  float* nsc = p.new_scores + (int64_t)bh * p.S;
  int32_t* kept = p.kept + (int64_t)bh * p.budget;
  if (tid == 0 && bh % p.KVH == 0) p.new_lengths[b] = m;

  constexpr int ROUND = kEvictThreads * E;
  const bool one = cand <= ROUND;  // every key stays in registers
  uint32_t key[E];
  auto load = [&](int base) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = base + tid * E + e;
      key[e] = j < cand ? evict_key(__ldg(sc + j)) : 0u;
    }
  };
  uint32_t thr = 0u;  // the largest key that at least `want` candidates reach
  if (want < cand) {  // want == cand keeps all: threshold 0
    if (one) load(0);
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = thr | (1u << bit);
      int c = 0;
      if (one) {
#pragma unroll
        for (int e = 0; e < E; ++e) c += key[e] >= trial;
      } else {
        for (int j = tid; j < cand; j += kEvictThreads) c += evict_key(__ldg(sc + j)) >= trial;
      }
      if (evict_block_sum(c, red, turn) >= want) thr = trial;
    }
  }
  // ties at the threshold that stay: the first `ties` of them
  int above = 0;
  for (int base = 0; base < cand; base += ROUND) {
    load(base);
    int c = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) c += key[e] > thr;
    above += evict_block_sum(c, red, turn);
  }
  const int ties = want - above;
  int tie_base = 0, out_base = 0;
  for (int base = 0; base < cand; base += ROUND) {
    load(base);
    int eq = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) eq += base + tid * E + e < cand && key[e] == thr;
    int sum;
    int tie = tie_base + evict_block_scan(eq, red, turn, &sum);
    tie_base += sum;
    unsigned keep = 0;
    int c = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = base + tid * E + e < cand;
      bool k = in && key[e] > thr;
      if (in && key[e] == thr) k = tie++ < ties;
      keep |= (unsigned)k << e;
      c += k;
    }
    int at = out_base + evict_block_scan(c, red, turn, &sum);
    out_base += sum;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (keep >> e & 1u) {
        const int j = base + tid * E + e;
        kept[at] = j;
        nsc[at] = sc[j];
        ++at;
      }
    }
  }
  for (int i = tid; i < r; i += kEvictThreads) {
    kept[want + i] = cand + i;
    nsc[want + i] = sc[cand + i];
  }
  for (int64_t i = m + tid; i < p.S; i += kEvictThreads) nsc[i] = 0.f;
  for (int i = m + tid; i < p.budget; i += kEvictThreads) kept[i] = -1;
}

// One CTA moves 32 kept cells of one sequence, all kv heads, K and V.
// P: the piece that rows are copied in (16 bytes where they allow it).
constexpr int kEvictCells = 32;
template <typename P>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  __shared__ int64_t s_new[kEvictCells];
  const int b = blockIdx.y, i0 = blockIdx.x * kEvictCells, tid = threadIdx.x;
  grid_dependency_wait();
  launch_dependents();
  const int n = evict_length(p, b);
  const int m = n < p.budget ? n : p.budget;
  if (i0 >= m) return;
  const int cells = m - i0 < kEvictCells ? m - i0 : kEvictCells;
  auto cell = [&](const int32_t* table, int width, int t) -> int64_t {
    const int pi = p.bs_shift >= 0 ? t >> p.bs_shift : t / p.block_size;
    const int page = pi < width ? __ldg(table + pi) : -1;
    if (page < 0 || (int64_t)page >= p.num_blocks) {
      raise_error(0x1u);
      return -1;
    }
    return (int64_t)page * p.block_size + (t - pi * p.block_size);
  };
  if (tid < cells) s_new[tid] = cell(p.new_tables + (int64_t)b * p.W2, p.W2, i0 + tid);
  __syncthreads();
  const int per_cell = p.KVH * p.row_pieces, total = cells * per_cell;
  P* pools[2] = {static_cast<P*>(p.k_pool), static_cast<P*>(p.v_pool)};
  for (int x = tid; x < total; x += 256) {
    const int i = x / per_cell, y = x % per_cell, h = y / p.row_pieces;
    const int64_t to = s_new[i];
    const int j = __ldg(p.kept + ((int64_t)b * p.KVH + h) * p.budget + i0 + i);
    const int64_t from = cell(p.tables + (int64_t)b * p.W, p.W, j);
    if (to < 0 || from < 0) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) pools[kv][to * per_cell + y] = pools[kv][from * per_cell + y];
  }
}

}  // namespace pdb
