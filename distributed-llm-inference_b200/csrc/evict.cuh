// Eviction from a paged cache by accumulated attention weight (sm_100a).
//
// Per (sequence, kv head) with n cached tokens, m = min(n, budget) stay: the
// last r = min(recent, m) tokens and, of the n - r others, the m - r of
// highest score (NaN lowest, equal scores by lowest index). They keep their
// order and go, K, V and score, to cells 0 .. m - 1 of new pages; every kv head
// keeps its own tokens, as a page holds each head's row separately.
//
// evict_select_kernel: one CTA per (sequence, kv head). Scores become 32-bit
// keys in the order of the floats (on a scale that is roughly logarithmic, so that
// scores of unlike magnitude spread evenly). The threshold is the largest key that
// at least m - r candidates reach: a histogram of the keys over kEvictBins equal
// steps of their range names the step that holds it, and the few keys of that step
// are ranked against each other. (Where one step holds too many keys to rank, or to
// list, the threshold's bits are found one by one, by counting. Counting alone, bit
// by bit over all keys, took 53 us for 48 x 8 heads of up to 8192 scores, bits past
// the twelfth over a list 34, this 29.) Counts per stripe of 32 scores, scanned
// once, number the ties and the kept tokens in index order.
// Rows are then copied in 16-byte pieces, bound by HBM: by the selecting CTA itself
// (its head's rows; one launch) where they are few, else by evict_move_kernel, which
// spreads a head over many CTAs (64 us for 421 MB, 6.5 TB/s).
#pragma once

#include <type_traits>

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
// Counts per (stripe, warp), stripe-major, to their exclusive prefix in place;
// returns their sum to every thread. Two barriers.
template <int E>
__device__ __forceinline__ int evict_scan_counts(int* counts) {
  static_assert(E * kEvictWarps <= 32 * E && kEvictWarps == 16, "16 E counts, one warp");
  __syncthreads();
  if (threadIdx.x < 32) {
    constexpr int PER = E / 2;  // 16 E counts over 32 lanes
    int v[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = counts[threadIdx.x * PER + i];
      mine += v[i];
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if ((int)threadIdx.x >= o) inc += y;
    }
    int run = inc - mine;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      counts[threadIdx.x * PER + i] = run;
      run += v[i];
    }
    if (threadIdx.x == 31) counts[16 * E] = inc;
  }
  __syncthreads();
  return counts[16 * E];
}

// Candidates per round of the CTA: E stripes of one per thread.
// First row (of the pool's cells x kv heads) of the cell of token t in `table`, -1
// without a page.
__device__ __forceinline__ int64_t evict_cell(const EvictParams& p, const int32_t* table, int width,
                                              int t) {
  const int pi = p.bs_shift >= 0 ? t >> p.bs_shift : t / p.block_size;
  const int page = pi < width ? __ldg(table + pi) : -1;
  if (page < 0 || (int64_t)page >= p.num_blocks) {
    raise_error(0x1u);
    return -1;
  }
  return ((int64_t)page * p.block_size + (t - pi * p.block_size)) * p.KVH;
}

constexpr int kEvictBins = 2048, kEvictList = 2048, kEvictRank = 512;
// P: the piece that rows are copied in, or void: another kernel copies them.
template <int E, typename P>
__global__ void __launch_bounds__(kEvictThreads, 3) evict_select_kernel(const EvictParams p) {
  __shared__ int red[2 * kEvictWarps];
  __shared__ int tie_counts[16 * E + 1], keep_counts[16 * E + 1], list_n, s_bin, s_higher;
  __shared__ uint32_t list[kEvictList], s_thr;
  __shared__ int bins[kEvictBins];
  int turn = 0;
  const int bh = blockIdx.x, b = bh / p.KVH, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  const bool one = cand <= ROUND;  // every score stays in registers
  uint32_t key[E];  // 0 (below every real key) past the candidates
  auto load = [&](int base) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = base + e * kEvictThreads + tid;
      key[e] = j < cand ? __float_as_uint(__ldg(sc + j)) : 0u;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      key[e] = base + e * kEvictThreads + tid < cand ? evict_key(__uint_as_float(key[e])) : 0u;
  };
  if (one) load(0);
  // what needs no selection
  for (int i = tid; i < r; i += kEvictThreads) {
    kept[want + i] = cand + i;
    nsc[want + i] = sc[cand + i];
  }
  for (int64_t i = m + tid; i < p.S; i += kEvictThreads) nsc[i] = 0.f;
  for (int i = m + tid; i < p.budget; i += kEvictThreads) kept[i] = -1;
  uint32_t thr = 0u;  // the largest key that at least `want` candidates reach
  if (want < cand && want > 0) {  // want == cand keeps all: threshold 0
    auto each = [&](auto&& fn) {  // every key of this thread; absent ones are 0
      if (one) {
#pragma unroll
        for (int e = 0; e < E; ++e) fn(key[e]);
      } else {
        for (int j = tid; j - tid < cand; j += kEvictThreads)
          fn(j < cand ? evict_key(__ldg(sc + j)) : 0u);
      }
    };
    // the keys' range, and its steps
    for (int i = tid; i < kEvictBins; i += kEvictThreads) bins[i] = 0;
    if (tid == 0) list_n = 0;
    uint32_t lo = 0xffffffffu, hi = 0u;
    each([&](uint32_t k) {
      if (k) lo = min(lo, k);
      hi = max(hi, k);
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      list[warp] = lo;
      list[kEvictWarps + warp] = hi;
    }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, list[lane & (kEvictWarps - 1)]);
    hi = __reduce_max_sync(0xffffffffu, list[kEvictWarps + (lane & (kEvictWarps - 1))]);
    const int width = 32 - __clz((int)(hi - lo));  // bits of the range
    const int shift = width > 11 ? width - 11 : 0;
    each([&](uint32_t k) {
      if (k) atomicAdd(&bins[(k - lo) >> shift], 1);  // whole numbers: any order
    });
    __syncthreads();
    // the step that holds the threshold: thread t sums 4 steps, highest first
    constexpr int PER = kEvictBins / kEvictThreads;
    int v[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = bins[kEvictBins - 1 - (tid * PER + i)];
      sum += v[i];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    int* r16 = red + turn * kEvictWarps;
    turn ^= 1;
    if (lane == 31) r16[warp] = inc;
    __syncthreads();
    int run = inc - sum;
#pragma unroll
    for (int w = 0; w < kEvictWarps; ++w)
      if (w < warp) run += r16[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (run < want && run + v[i] >= want) {
        s_bin = kEvictBins - 1 - (tid * PER + i);
        s_higher = run;
      }
      run += v[i];
    }
    __syncthreads();
    const int bin = s_bin, higher = s_higher, need = want - higher;
    const uint32_t base = lo + ((uint32_t)bin << shift), steps = (1u << shift) - 1u;
    // that step's keys
    each([&](uint32_t k) {
      const bool in = k >= base && k - base <= steps;
      const unsigned mask = __ballot_sync(0xffffffffu, in);
      int at = 0;
      if (lane == 0 && mask) at = atomicAdd(&list_n, __popc(mask));  // order does not matter
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(mask & ((1u << lane) - 1));
      if (in && at < kEvictList) list[at] = k;
    });
    __syncthreads();
    const int ln = list_n;
    if (ln <= kEvictRank) {
      if (tid < ln) {
        const uint32_t k = list[tid];
        int above = 0, same = 0;
        for (int x = 0; x < ln; ++x) {
          above += list[x] > k;
          same += list[x] == k;
        }
        if (above < need && above + same >= need) s_thr = k;  // every such thread: one value
      }
      __syncthreads();
      thr = s_thr;
    } else {
      thr = base;
      for (int bit = shift - 1; bit >= 0; --bit) {
        const uint32_t trial = base + ((thr - base) | (1u << bit));
        int c = 0;
        if (ln <= kEvictList) {
          for (int j = tid; j < ln; j += kEvictThreads) c += list[j] >= trial;
          c = evict_block_sum(c, red, turn) + higher;
        } else {
          each([&](uint32_t k) { c += k >= trial; });
          c = evict_block_sum(c, red, turn);
        }
        if (c >= want) thr = trial;
      }
    }
  } else if (want == 0) {
    thr = 0xffffffffu;  // none of the candidates
  }
  // ties at the threshold that stay: the first `ties` of them
  int above = 0;
  if (one) {
#pragma unroll
    for (int e = 0; e < E; ++e) above += key[e] > thr;
  } else {
    for (int j = tid; j < cand; j += kEvictThreads) above += evict_key(__ldg(sc + j)) > thr;
  }
  const int ties = want - evict_block_sum(above, red, turn);
  int tie_base = 0, out_base = 0;
  const unsigned below = (1u << lane) - 1;
  for (int base = 0; base < cand; base += ROUND) {
    if (!one) load(base);
    // ballots are taken again where they are needed: kept, they would cost 32
    // registers and the third CTA per SM
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned eq = __ballot_sync(0xffffffffu, key[e] == thr && key[e] != 0u);
      if (lane == 0) tie_counts[e * kEvictWarps + warp] = __popc(eq);
    }
    const int tie_sum = evict_scan_counts<E>(tie_counts);
    unsigned mine = 0;  // bit e: this thread's key of stripe e stays
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool tie = key[e] == thr && key[e] != 0u;
      const unsigned eq = __ballot_sync(0xffffffffu, tie);
      const int rank = tie_base + tie_counts[e * kEvictWarps + warp] + __popc(eq & below);
      const bool stays = key[e] > thr || (tie && rank < ties);
      mine |= (unsigned)stays << e;
      const unsigned keep = __ballot_sync(0xffffffffu, stays);
      if (lane == 0) keep_counts[e * kEvictWarps + warp] = __popc(keep);
    }
    const int keep_sum = evict_scan_counts<E>(keep_counts);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool stays = mine >> e & 1u;
      const unsigned keep = __ballot_sync(0xffffffffu, stays);
      if (stays) {
        const int at = out_base + keep_counts[e * kEvictWarps + warp] + __popc(keep & below);
        const int j = base + e * kEvictThreads + tid;
        kept[at] = j;
        nsc[at] = __ldg(sc + j);
      }
    }
    tie_base += tie_sum;
    out_base += keep_sum;
  }
  if constexpr (!std::is_void<P>::value) {
    // this head's rows, kEvictThreads at a time: their cells, then their pieces with
    // eight loads in flight per thread
    __shared__ int64_t s_from[kEvictThreads], s_to[kEvictThreads];
    const int h = bh - b * p.KVH, rp = p.row_pieces;
    P* kp = static_cast<P*>(p.k_pool);
    P* vp = static_cast<P*>(p.v_pool);
    constexpr int U = 4;
    for (int i0 = 0; i0 < m; i0 += kEvictThreads) {
      __syncthreads();  // `kept` is written; the cells of the rows before are read
      if (i0 + tid < m) {
        s_from[tid] = evict_cell(p, p.tables + (int64_t)b * p.W, p.W, kept[i0 + tid]);
        s_to[tid] = evict_cell(p, p.new_tables + (int64_t)b * p.W2, p.W2, i0 + tid);
      }
      __syncthreads();
      const int total = (m - i0 < kEvictThreads ? m - i0 : kEvictThreads) * rp;
      for (int x0 = tid; x0 < total; x0 += kEvictThreads * U) {
        P kx[U], vx[U];
        int64_t to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int x = x0 + u * kEvictThreads;
          to[u] = -1;
          if (x < total) {
            const int i = x / rp, c = x - i * rp;
            const int64_t from = s_from[i], dst = s_to[i];
            if (from >= 0 && dst >= 0) {
              to[u] = (dst + h) * rp + c;
              kx[u] = kp[(from + h) * rp + c];
              vx[u] = vp[(from + h) * rp + c];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (to[u] >= 0) {
            kp[to[u]] = kx[u];
            vp[to[u]] = vx[u];
          }
      }
    }
  }
}

// One CTA moves 32 kept cells of up to 8 kv heads of one sequence, K and V: the
// cells are looked up once into shared memory, then the pieces of their rows are
// copied with eight loads in flight per thread.
// P: the piece that rows are copied in (16 bytes where they allow it).
constexpr int kEvictCells = 32, kEvictHeads = 8;
template <typename P>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  __shared__ int64_t s_from[kEvictCells * kEvictHeads], s_new[kEvictCells];
  const int b = blockIdx.y, i0 = blockIdx.x * kEvictCells, h0 = blockIdx.z * kEvictHeads;
  const int tid = threadIdx.x;
  grid_dependency_wait();
  launch_dependents();
  const int n = evict_length(p, b);
  const int m = n < p.budget ? n : p.budget;
  if (i0 >= m) return;
  const int cells = m - i0 < kEvictCells ? m - i0 : kEvictCells;
  const int heads = p.KVH - h0 < kEvictHeads ? p.KVH - h0 : kEvictHeads;
  {  // 256 = 32 cells x 8 heads: neighbouring threads take neighbouring kept tokens
    const int i = tid % kEvictCells, h = tid / kEvictCells;
    if (i < cells && h < heads) {
      const int j = __ldg(p.kept + ((int64_t)b * p.KVH + h0 + h) * p.budget + i0 + i);
      s_from[tid] = evict_cell(p, p.tables + (int64_t)b * p.W, p.W, j);
    }
    if (h == 0 && i < cells) s_new[i] = evict_cell(p, p.new_tables + (int64_t)b * p.W2, p.W2, i0 + i);
  }
  __syncthreads();
  const int rp = p.row_pieces, per_cell = heads * rp, total = cells * per_cell;
  P* kp = static_cast<P*>(p.k_pool);
  P* vp = static_cast<P*>(p.v_pool);
  constexpr int U = 4;
  for (int x0 = tid; x0 < total; x0 += 256 * U) {
    P kx[U], vx[U];
    int64_t to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = x0 + u * 256;
      to[u] = -1;
      if (x < total) {
        const int i = x / per_cell, y = x - i * per_cell, h = y / rp, c = y - h * rp;
        const int64_t from = s_from[h * kEvictCells + i], dst = s_new[i];
        if (from >= 0 && dst >= 0) {
          const int64_t at = (from + h0 + h) * rp + c;
          to[u] = (dst + h0 + h) * rp + c;
          kx[u] = kp[at];
          vx[u] = vp[at];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] >= 0) {
        kp[to[u]] = kx[u];
        vp[to[u]] = vx[u];
      }
  }
}

}  // namespace pdb
