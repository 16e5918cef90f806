// Attention of a batch whose sequences share a long prefix (sm_100a).
//
// Sequence b brings T query tokens (n_b = counts[b] of them real), which see
// the prefix's P cached tokens and their own: token t sees own tokens
// 0 .. lengths[b] - n_b + t. The softmax over both parts is a join of partial
// softmaxes: with s_j the logits in base 2 (log2(e) / sqrt(D) folded in), any
// set X of keys gives
//   m_X = max s_j,  l_X = sum 2^(s_j - m_X),  O_X = sum 2^(s_j - m_X) v_j
// and disjoint sets join by m = max m_X, l = sum 2^(m_X - m) l_X, the same for
// O; the output is O / l. So the prefix is one key set for ALL rows of a kv
// head (B T G of them: its K and V are read once per row tile, not once per
// sequence) and a sequence's own tokens are another for its T G rows.
//
// Rows of a kv head are numbered r = (b T + t) G + g; the rows of sequence b
// are [b T G, (b + 1) T G). A partial is (m, l) and O of some rows over a key
// range, in FP32: ml [..] float2, o [..][D]. The prefix's partials and those of
// own tokens are two sets (PartSet), each written by one of these kernels:
//   * the kernels here and the TF32 kernel: fixed key ranges ("slots") of every row,
//     part index = slot * rows + global row (b T + t) H + h;
//   * the tensor-core kernels: work in units (64- or 128-key tiles of a segment
//     of rows), cut into one contiguous range per CTA; CTA c's piece of segment
//     s is stored as piece s + c (distinct for distinct pieces, as each step to
//     the next piece raises s, c or both), part index = piece * R + row of the
//     segment. The pieces of a segment are those of consecutive CTAs; the first
//     and the last of them are noted in `dir`.
// Either way a row's partials are evenly spaced: prefix_join_kernel joins them.
#pragma once

#include <type_traits>

#include "attention.cuh"

namespace pdb {

// `units` cut into one range per CTA, lengths equal up to one; CTAs that share
// them each have at least one, so the pieces of a segment are those of
// consecutive CTAs. First unit of CTA c (of `ctas`; c = ctas: the end).
__host__ __device__ __forceinline__ int unit_ctas(int units, int grid) {
  return units < grid ? units : grid;
}
__device__ __forceinline__ int unit_begin(int c, int units, int ctas) {
  if (c >= ctas) return units;
  const unsigned per = (unsigned)units / (unsigned)ctas, more = (unsigned)units - per * ctas;
  return c * (int)per + (c < (int)more ? c : (int)more);
}

enum : int { kPartNone = 0, kPartSlots = 1, kPartUnits = 2 };

struct PartSet {
  float2* ml;
  float* o;
  int2* dir;          // kPartUnits: [segments of all sequences and kv heads] first, last CTA
  int kind;
  int slots, chunk;   // kPartSlots: key ranges [i * chunk, (i + 1) * chunk)
  int R;              // kPartUnits: rows of a segment
  int half;           //   tokens of its first R / 2 rows (two query tiles), or 0: rows are dense
  int segments;       //   segments per (sequence,) kv head
  int first;          //   index of the first segment
  int grid;           //   CTAs that share the units
};

struct PrefixParams {
  const void* q;                // [B, T, H, D]
  const void* k_pool;           // [N, bs, KVH, D]
  const void* v_pool;
  const int32_t* prefix_table;  // [ceil(P / bs)]
  const int32_t* tables;        // [B, W]
  const int32_t* lengths;       // [B]
  const int32_t* counts;        // [B] or NULL (all T)
  void* out;                    // [B, T, H, D]
  PartSet prefix, own;          // partials
  float* lse;                   // [rows] base-2 log of the softmax's denominator (scores only)
  float* logits;                // [B, KVH, logits_width, T G] base-2 logits of own tokens, or NULL
  const float* scores;          // [B, KVH, scores_width]
  float* scores_out;
  int64_t num_blocks, rows, logits_width, scores_width;
  int B, T, H, KVH, G, D;
  int block_size, bs_shift, table_width;
  int prefix_length, max_length;
  float scale_log2;
  int beside;  // the own-token kernel follows this call's prefix kernel, whose CTAs let it start
               // only once all work before it was complete: it waits for it at its end
};

// Tokens, length and first visible row of sequence b, clamped to what the
// tables hold (out-of-range values raise an error bit).
__device__ __forceinline__ void prefix_sequence(const PrefixParams& p, int b, int& n, int& count) {
  n = __ldg(p.lengths + b);
  count = p.counts ? __ldg(p.counts + b) : p.T;
  if (n < 0 || n > p.max_length || count < 0 || count > p.T) {
    raise_error(0x2u);
    n = n < 0 ? 0 : (n > p.max_length ? p.max_length : n);
    count = count < 0 ? 0 : (count > p.T ? p.T : count);
  }
}
// Own keys [0, limit) that token t sees; -1 for a token that is not real.
__device__ __forceinline__ int prefix_limit(int n, int count, int t) {
  if (t >= count) return -1;
  const int lim = n - count + t + 1;
  return lim < 0 ? 0 : lim;
}

// Pool row of token `tok` of a page list, or -1 (page out of range).
__device__ __forceinline__ int64_t prefix_cell(const PrefixParams& p, const int32_t* table,
                                               int width, int tok) {
  const int pi = p.bs_shift >= 0 ? tok >> p.bs_shift : tok / p.block_size;
  const int page = pi < width ? __ldg(table + pi) : -1;
  if (page < 0 || (int64_t)page >= p.num_blocks) {
    raise_error(0x1u);
    return -1;
  }
  return (int64_t)page * p.block_size + (tok - pi * p.block_size);
}

// The rows and keys of a CTA of the kernels with slots, by blockIdx.x: the prefix's
// (row tile, range) pairs, or own (sequence, row tile, range) triples.
struct SpanTile {
  int slot, b;           // b: sequence, or -1 (the prefix)
  int k0, k1;            // keys; none: k0 >= k1
  int n, count;          // of the sequence
  int r0, rend, token0;  // rows [r0, rend) as tokens from token0, heads inner
  const int32_t* table;
  int width;
};
__device__ __forceinline__ SpanTile span_tile(const PrefixParams& p, const PartSet& set,
                                              bool prefix, int own_tiles, int rt) {
  SpanTile t;
  int x = blockIdx.x;
  t.slot = x % set.slots;
  x /= set.slots;
  t.count = 0;
  if (prefix) {
    t.b = -1;
    t.r0 = x * rt;
    t.token0 = 0;
    t.rend = p.B * p.T * p.G;
    t.n = p.prefix_length;
    t.table = p.prefix_table;
    t.width = (p.prefix_length + p.block_size - 1) / p.block_size;
  } else {
    t.b = x / own_tiles;
    prefix_sequence(p, t.b, t.n, t.count);
    t.r0 = x % own_tiles * rt;
    t.token0 = t.b * p.T;
    t.rend = p.T * p.G;
    t.table = p.tables + (int64_t)t.b * p.table_width;
    t.width = p.table_width;
  }
  t.k0 = t.slot * set.chunk;
  t.k1 = t.k0 + set.chunk < t.n ? t.k0 + set.chunk : t.n;
  return t;
}

// ---- spans on the FP32 pipes (any type, head_dim <= DP, block size, alignment) --
// One CTA per (row tile of RT, kv head, key range), keys in tiles of KT staged
// in shared memory as FP32, two tiles in flight. Products and sums are FP32
// throughout. A thread holds RPT rows x KPT
// keys of S and RPT rows x OPT groups of 4 dims of O, everything read from shared
// memory in 16-byte pieces. Such a read takes the SM four cycles whatever it
// reads, so the reads per multiply-add bound the kernel: 8 per 64 with 4 x 4 keys and
// rows a thread (head_dim 128, 64 rows), 6 per 32 with 2 x 4. Grid: x = the prefix's
// (row tile, range) pairs, or own (sequence, row tile, chunk) triples; y = kv head.
template <int DP, int RT>
struct PrefixSimt {
  static constexpr int NT = 128;
  static constexpr int KT = DP == 64 ? 64 : DP == 128 ? 32 : 16;
  static constexpr int LD = DP + 4;          // padded row of Q and K: rows 4 banks apart
  static constexpr int RPT = RT == 64 ? 4 : RT == 32 ? 2 : 1;
  static constexpr int TPR = NT * RPT / RT;  // threads that share a row: 8 or 16
  static constexpr int KPT = KT / TPR;       // keys per thread of S
  static constexpr int OPT = DP / 4 / TPR;   // groups of 4 dims per thread of O
  static constexpr int LP = KT + 4;          // padded row of P
  static constexpr size_t SMEM =
      (size_t)(RT * LD + 2 * KT * LD + 2 * KT * DP + RT * LP) * sizeof(float);
};

template <typename T, int DP, int RT>
__global__ void __launch_bounds__(PrefixSimt<DP, RT>::NT)
prefix_simt_kernel(const PrefixParams p, int prefix_tiles, int own_tiles) {
  using C = PrefixSimt<DP, RT>;
  constexpr int NT = C::NT, KT = C::KT, LD = C::LD, RPT = C::RPT, TPR = C::TPR, KPT = C::KPT,
                OPT = C::OPT, LP = C::LP;
  extern __shared__ __align__(16) float smem_f[];
  float* sq = smem_f;              // [RT][LD]
  float* sk = sq + RT * LD;        // [2][KT][LD]
  float* sv = sk + 2 * KT * LD;    // [2][KT][DP]
  float* sp = sv + 2 * KT * DP;    // [RT][LP]
  const int tid = threadIdx.x, h = blockIdx.y, D = p.D, G = p.G;
  const bool prefix = prefix_tiles > 0, beside = !prefix && p.beside;
  if (!beside) grid_dependency_wait();
  launch_dependents();

  const PartSet& set = prefix ? p.prefix : p.own;
  const SpanTile t = span_tile(p, set, prefix, own_tiles, RT);
  const int slot = t.slot, b = t.b, k0 = t.k0, k1 = t.k1, n = t.n, count = t.count,
            width = t.width, r0 = t.r0, rend = t.rend;
  const int32_t* table = t.table;
  if (k0 >= k1) {
    if (beside) grid_dependency_wait();
    return;
  }
  auto global_row = [&](int row) {  // of q and out
    return (int64_t)(t.token0 + row / G) * p.H + (int64_t)h * G + row % G;
  };
  const T* q = static_cast<const T*>(p.q);
  const T* kp = static_cast<const T*>(p.k_pool);
  const T* vp = static_cast<const T*>(p.v_pool);

  // stage keys [t0, t0 + KT) into buffer `buf`; rows past the range: zeros, so that a
  // zero weight stays zero
  auto stage = [&](int t0, int buf) {
    float* dk = sk + buf * KT * LD;
    float* dv = sv + buf * KT * DP;
#pragma unroll 4
    for (int i = tid; i < KT * D; i += NT) {
      const int j = i / D, d = i % D;
      const int64_t cell = t0 + j < k1 ? prefix_cell(p, table, width, t0 + j) : -1;
      const int64_t at = (cell * p.KVH + h) * D + d;
      dk[j * LD + d] = cell < 0 ? 0.f : Elem<T>::to_f(kp[at]);
      dv[j * DP + d] = cell < 0 ? 0.f : Elem<T>::to_f(vp[at]);
    }
  };
  if (D < DP) {  // dims past D are never staged
    for (int i = tid; i < 2 * KT * LD; i += NT) sk[i] = 0.f;
    for (int i = tid; i < 2 * KT * DP; i += NT) sv[i] = 0.f;
    __syncthreads();
  }
  stage(k0, 0);
#pragma unroll 8
  for (int i = tid; i < RT * DP; i += NT) {
    const int r = i / DP, d = i % DP;
    float v = 0.f;
    if (r0 + r < rend && d < D) v = Elem<T>::to_f(q[global_row(r0 + r) * D + d]);
    sq[r * LD + d] = v;
  }
  const int rg = tid / TPR, part = tid % TPR;  // rows rg RPT .., keys and dims part, part + TPR, ..
  int limit[RPT];  // keys [0, limit) are seen
  float m[RPT], l[RPT], acc[RPT][OPT][4];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int row = r0 + rg * RPT + r;
    limit[r] = prefix ? k1 : row < rend ? prefix_limit(n, count, row / G) : -1;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < OPT; ++i) acc[r][i][0] = acc[r][i][1] = acc[r][i][2] = acc[r][i][3] = 0.f;
  }
  float* logits = p.logits && b >= 0
                      ? p.logits + ((int64_t)b * p.KVH + h) * p.logits_width * p.T * G
                      : nullptr;

  int buf = 0;
  for (int t0 = k0; t0 < k1; t0 += KT, buf ^= 1) {
    if (t0 + KT < k1) stage(t0 + KT, buf ^ 1);
    __syncthreads();
    const float* ck = sk + buf * KT * LD;
    const float* cv = sv + buf * KT * DP;
    float s[RPT][KPT];
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
      for (int i = 0; i < KPT; ++i) s[r][i] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 a[RPT];
#pragma unroll
      for (int r = 0; r < RPT; ++r)
        a[r] = *reinterpret_cast<const float4*>(sq + (rg * RPT + r) * LD + d);
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(ck + (part + i * TPR) * LD + d);
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          s[r][i] = fmaf(a[r].x, y.x, s[r][i]);
          s[r][i] = fmaf(a[r].y, y.y, s[r][i]);
          s[r][i] = fmaf(a[r].z, y.z, s[r][i]);
          s[r][i] = fmaf(a[r].w, y.w, s[r][i]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      const int row = r0 + rg * RPT + r;
      float mt = -INFINITY;
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const int key = t0 + part + i * TPR;
        const bool seen = key < limit[r] && key < k1;
        s[r][i] = seen ? s[r][i] * p.scale_log2 : -INFINITY;
        if (logits && seen) logits[(int64_t)key * p.T * G + row] = s[r][i];
        mt = fmaxf(mt, s[r][i]);
      }
#pragma unroll
      for (int o = 1; o < TPR; o <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      const float mn = fmaxf(m[r], mt);
      const float alpha = mn == -INFINITY ? 1.f : exp2f(m[r] - mn);  // m = -inf: 0
      const float ref = mn == -INFINITY ? 0.f : mn;
      l[r] *= alpha;
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const float w = exp2f(s[r][i] - ref);
        l[r] += w;
        sp[(rg * RPT + r) * LP + part + i * TPR] = w;
      }
      m[r] = mn;
#pragma unroll
      for (int i = 0; i < OPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][i][e] *= alpha;
    }
    __syncwarp();  // a row's threads are in one warp
    // keys that this row must not see have weight 0, and a v that may be anything: in
    // the tiles that hold such keys a zero weight skips its key
    const bool mask = !prefix && t0 + KT > n - count + 1;
#pragma unroll 2
    for (int j = 0; j < KT; j += 4) {
      float4 w4[RPT];
#pragma unroll
      for (int r = 0; r < RPT; ++r)
        w4[r] = *reinterpret_cast<const float4*>(sp + (rg * RPT + r) * LP + j);
#pragma unroll
      for (int jj = 0; jj < 4; ++jj)
#pragma unroll
        for (int i = 0; i < OPT; ++i) {
          const float4 y =
              *reinterpret_cast<const float4*>(cv + (j + jj) * DP + (part + i * TPR) * 4);
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const float w = jj == 0 ? w4[r].x : jj == 1 ? w4[r].y : jj == 2 ? w4[r].z : w4[r].w;
            if (mask && w == 0.f) continue;
            acc[r][i][0] = fmaf(w, y.x, acc[r][i][0]);
            acc[r][i][1] = fmaf(w, y.y, acc[r][i][1]);
            acc[r][i][2] = fmaf(w, y.z, acc[r][i][2]);
            acc[r][i][3] = fmaf(w, y.w, acc[r][i][3]);
          }
        }
    }
    __syncthreads();  // the buffer may be staged again
  }
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
    const int row = r0 + rg * RPT + r;
    if (row >= rend) continue;
    const int64_t at = (int64_t)slot * p.rows + global_row(row);
    if (part == 0) set.ml[at] = make_float2(m[r], l[r]);
#pragma unroll
    for (int i = 0; i < OPT; ++i) {
      const int d = (part + i * TPR) * 4;
      if (d + 4 <= D && D % 4 == 0)
        *reinterpret_cast<float4*>(set.o + at * D + d) =
            make_float4(acc[r][i][0], acc[r][i][1], acc[r][i][2], acc[r][i][3]);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) set.o[at * D + d + e] = acc[r][i][e];
    }
  }
  if (beside) grid_dependency_wait();
}

// ---- spans of few rows on the FP32 pipes ------------------------------------------
// FP32 with head_dim DP and at most R = 4 or 8 rows per sequence (T G), 16-byte pieces:
// decode steps, bound by HBM if shared memory is read little enough. Eight lanes
// share a key and hold the queries' dims of their slice in registers for all R rows,
// so a key's row costs DP / 32 reads per lane for R DP / 8 multiply-adds; a
// butterfly that halves the rows at each step leaves lane i of the eight with row
// i's logit. Each warp takes 8 keys of a 32-key tile with its own running maximum
// and sum, and DP / 32 dims of all R rows of O per lane; the four warps are joined at
// the end. Three tiles in flight by cp.async, pages looked up one key per lane.
// (8 x 8 kv heads of 2048 to 8192 keys, head_dim 128: 171 us with the kernel above,
// whose 3 reads per 8 multiply-adds keep shared memory busy, 85 here with the join.)
template <int DP, int R>
struct PrefixFew {
  static constexpr int NT = 128, KT = 32, STAGES = 3;
  static constexpr int SL = DP / 32;  // 16-byte pieces of a lane's slice of a row
  static constexpr int VL = DP / 32;  // dims of O per lane
  static constexpr int STAGE = 2 * KT * DP;
  static constexpr size_t SMEM = (size_t)(STAGES * STAGE + 4 * 8 * R + 4 * R * 2) * sizeof(float);
  static_assert(4 * R * DP <= STAGE, "join buffer fits a stage");
};

template <int DP, int R>
__global__ void __launch_bounds__(PrefixFew<DP, R>::NT, 2)
prefix_few_kernel(const PrefixParams p) {
  using C = PrefixFew<DP, R>;
  constexpr int KT = C::KT, STAGES = C::STAGES, SL = C::SL, VL = C::VL, NT = C::NT;
  extern __shared__ __align__(16) float smem_f[];
  float* sp = smem_f + STAGES * C::STAGE;  // [4 warps][8 keys][R]
  float* sm = sp + 4 * 8 * R;              // [4][R] maxima, then [4][R] sums
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y, G = p.G;
  const int sub = lane & 7, kq = lane >> 3, row = sub % R;
  if (!p.beside) grid_dependency_wait();
  launch_dependents();
  const int slot = blockIdx.x % p.own.slots, b = blockIdx.x / p.own.slots;
  int n, count;
  prefix_sequence(p, b, n, count);
  const int k0 = slot * p.own.chunk, k1 = k0 + p.own.chunk < n ? k0 + p.own.chunk : n;
  if (k0 >= k1) {
    if (p.beside) grid_dependency_wait();
    return;
  }
  const int rows = p.T * G;
  const int32_t* table = p.tables + (int64_t)b * p.table_width;
  const float* kp = static_cast<const float*>(p.k_pool) + (int64_t)h * DP;
  const float* vp = static_cast<const float*>(p.v_pool) + (int64_t)h * DP;
  auto cell_of = [&](int key) -> int64_t {
    return key < k1 ? prefix_cell(p, table, p.table_width, key) : -1;
  };
  auto stage = [&](int st, int64_t cell) {  // lane j holds the cell of key j
    float* dk = smem_f + st * C::STAGE;
    float* dv = dk + KT * DP;
    constexpr int PIECES = DP / 4, PER = 32 / PIECES > 0 ? 32 / PIECES : 1;  // rows per warp read
#pragma unroll
    for (int i = 0; i < KT / (4 * PER); ++i) {
      const int j = (i * 4 + warp) * PER + (PIECES < 32 ? lane / PIECES : 0);
      const int64_t at = __shfl_sync(0xffffffffu, cell, j);
      const int c = (PIECES < 32 ? lane % PIECES : lane) * 4;
      const int64_t e = at < 0 ? 0 : at * p.KVH * DP + c;
      cp_async16(dk + j * DP + c, kp + e, at >= 0);  // no page, past the end: zeros
      cp_async16(dv + j * DP + c, vp + e, at >= 0);
    }
  };
  int64_t cell = cell_of(k0 + lane);
  int next = k0;
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) {
    if (next < k1) {
      stage(st, cell);
      next += KT;
      cell = cell_of(next + lane);
    }
    cp_async_commit();
  }
  // this lane's slice of the queries
  float4 q[R][SL];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < SL; ++c) {
      q[r][c] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) {
        const float* src = static_cast<const float*>(p.q) +
                           ((int64_t)(b * p.T + r / G) * p.H + (int64_t)h * G + r % G) * DP +
                           (c * 8 + sub) * 4;
        q[r][c] = make_float4(src[0] * p.scale_log2, src[1] * p.scale_log2,
                              src[2] * p.scale_log2, src[3] * p.scale_log2);
      }
    }
  const int limit = row < rows ? prefix_limit(n, count, row / G) : -1;
  float* logits = p.logits && row < rows && sub < R
                      ? p.logits + ((int64_t)b * p.KVH + h) * p.logits_width * rows + row
                      : nullptr;
  float m = -INFINITY, l = 0.f, acc[R][VL];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < VL; ++i) acc[r][i] = 0.f;
  float* pw = sp + warp * 8 * R;

  int st = 0;
  for (int t0 = k0; t0 < k1; t0 += KT, st = st + 1 == STAGES ? 0 : st + 1) {
    cp_async_wait<STAGES - 2>();
    __syncthreads();  // this tile landed for all; the stage before it is read
    if (next < k1) {
      stage(st == 0 ? STAGES - 1 : st - 1, cell);
      next += KT;
      cell = cell_of(next + lane);
    }
    cp_async_commit();
    const float* ck = smem_f + st * C::STAGE + warp * 8 * DP;
    const float* cv = ck + KT * DP;
    if (t0 + warp * 8 >= k1) continue;  // none of this warp's keys (the barriers are above)
    float s[2];
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      float x[R];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = 0.f;
#pragma unroll
      for (int c = 0; c < SL; ++c) {
        const float4 y =
            *reinterpret_cast<const float4*>(ck + (pass * 4 + kq) * DP + (c * 8 + sub) * 4);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[r] = fmaf(q[r][c].x, y.x, x[r]);
          x[r] = fmaf(q[r][c].y, y.y, x[r]);
          x[r] = fmaf(q[r][c].z, y.z, x[r]);
          x[r] = fmaf(q[r][c].w, y.w, x[r]);
        }
      }
      // rows halved, partners added: lane `sub` ends with row sub % R
#pragma unroll
      for (int half = R / 2; half; half >>= 1) {
        const bool up = sub & half;
#pragma unroll
        for (int r = 0; r < half; ++r) {
          const float give = up ? x[r] : x[r + half];
          x[r] = (up ? x[r + half] : x[r]) + __shfl_xor_sync(0xffffffffu, give, half);
        }
      }
      if constexpr (R == 4) x[0] += __shfl_xor_sync(0xffffffffu, x[0], 4);
      const int key = t0 + warp * 8 + pass * 4 + kq;
      const bool seen = key < limit && key < k1;
      if (logits && seen) logits[(int64_t)key * rows] = x[0];
      s[pass] = seen ? x[0] : -INFINITY;
    }
    float top = fmaxf(s[0], s[1]);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    float alpha = 1.f;
    if (top > m) {
      alpha = exp2f(m - top);  // m = -inf: 0
      m = top;
    }
    if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float a = __shfl_sync(0xffffffffu, alpha, r);
#pragma unroll
        for (int i = 0; i < VL; ++i) acc[r][i] *= a;
      }
    }
    const float ref = m == -INFINITY ? 0.f : m;
    const float w0 = exp2f(s[0] - ref), w1 = exp2f(s[1] - ref);
    l = l * alpha + (w0 + w1);
    __syncwarp();  // the weights of the tile before are read
    if (sub < R) {
      pw[kq * R + row] = w0;
      pw[(4 + kq) * R + row] = w1;
    }
    __syncwarp();
    // keys that a row must not see have weight 0, and a v that may be anything
    const bool mask = t0 + KT > n - count + 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float w[R], v[VL];
#pragma unroll
      for (int r = 0; r < R; r += 4) {
        const float4 y = *reinterpret_cast<const float4*>(pw + k * R + r);
        w[r] = y.x; w[r + 1] = y.y; w[r + 2] = y.z; w[r + 3] = y.w;
      }
      if constexpr (VL == 4) {
        const float4 y = *reinterpret_cast<const float4*>(cv + k * DP + lane * 4);
        v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
      } else {
        const float2 y = *reinterpret_cast<const float2*>(cv + k * DP + lane * 2);
        v[0] = y.x; v[1] = y.y;
      }
      if (mask) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (w[r] != 0.f)
#pragma unroll
            for (int i = 0; i < VL; ++i) acc[r][i] = fmaf(w[r], v[i], acc[r][i]);
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < VL; ++i) acc[r][i] = fmaf(w[r], v[i], acc[r][i]);
      }
    }
  }
  // join of the four warps
  l += __shfl_xor_sync(0xffffffffu, l, 8);
  l += __shfl_xor_sync(0xffffffffu, l, 16);
  if (lane < R) {
    sm[warp * R + lane] = m;
    sm[4 * R + warp * R + lane] = l;
  }
  cp_async_wait<0>();
  __syncthreads();  // every tile is read: the first stage takes the join
  float* jb = smem_f;  // [4][R][DP]
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float t = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) t = fmaxf(t, sm[w * R + r]);
    const float mine = sm[warp * R + r], a = mine == -INFINITY ? 0.f : exp2f(mine - t);
#pragma unroll
    for (int i = 0; i < VL; ++i) jb[(warp * R + r) * DP + lane * VL + i] = acc[r][i] * a;
  }
  __syncthreads();
  for (int x = tid; x < rows * DP; x += NT) {
    const int r = x / DP, d = x - r * DP;
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o += jb[(w * R + r) * DP + d];
    const int64_t at = (int64_t)slot * p.rows + (int64_t)(b * p.T + r / G) * p.H +
                       (int64_t)h * G + r % G;
    p.own.o[at * DP + d] = o;
    if (d == 0) {
      float t = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) t = fmaxf(t, sm[w * R + r]);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        sum += sm[4 * R + w * R + r] * (sm[w * R + r] == -INFINITY ? 0.f : exp2f(sm[w * R + r] - t));
      p.own.ml[at] = make_float2(t, sum);
    }
  }
  if (p.beside) grid_dependency_wait();
}

// ---- join of the partials -----------------------------------------------------
// A row's partials in one set: part indices at, at + step, .. (count of them).
struct PartRange {
  int64_t at, step;
  int count;
};
// Token t (of those that share segments), head g of the group: the row of its
// segment; `seg` becomes the segment's index (it comes in as that of the first).
__device__ __forceinline__ PartRange prefix_parts(const PartSet& s, int seg, int t, int g, int G) {
  int lr;
  if (s.half) {  // two query tiles of R / 2 rows, each with a remainder of unused rows
    const int x = t / s.half, in = t - x * s.half;
    seg += x >> 1;
    lr = (x & 1) * (s.R / 2) + in * G + g;
  } else {
    const int r = t * G + g, x = r / s.R;
    seg += x;
    lr = r - x * s.R;
  }
  const int2 c = s.dir[seg];
  return PartRange{(int64_t)(seg + c.x) * s.R + lr, s.R, c.y - c.x + 1};
}

// sum 2^(s_j - m) v_j of one row in plain FP32, key by key, four dims per lane and LPR lanes
// of a warp (`mask`): for rows whose sum came out as a NaN although their logits have none. The
// tensor cores take a weight as two FP16 numbers, and where one of them is 0 (a weight that
// is exact in FP16, or too small for it) an infinite v_j gives 0 * inf. Rare and slow; not inlined, so
// that the join's own code stays short.
template <int LPR>
__device__ __noinline__ float4 prefix_row_plain(const PrefixParams& p, int64_t row, int b, int h,
                                                int limit, float m, unsigned mask) {
  const int lane = threadIdx.x % LPR, D = p.D;
  const bool in = 4 * lane < D;
  float q[4] = {}, acc[4] = {};
  if (in)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = __half2float(static_cast<const __half*>(p.q)[row * D + 4 * lane + i]) * p.scale_log2;
  for (int set = 0; set < 2; ++set) {
    const int32_t* table = set ? p.tables + (int64_t)b * p.table_width : p.prefix_table;
    const int width = set ? p.table_width : (p.prefix_length + p.block_size - 1) / p.block_size;
    const int keys = set ? limit : p.prefix_length;
    for (int j = 0; j < keys; ++j) {
      const int64_t cell = prefix_cell(p, table, width, j);
      const int64_t at = (cell * p.KVH + h) * D + 4 * lane;
      float s = 0.f, v[4] = {};
      if (in && cell >= 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s = fmaf(q[i], __half2float(static_cast<const __half*>(p.k_pool)[at + i]), s);
          v[i] = __half2float(static_cast<const __half*>(p.v_pool)[at + i]);
        }
#pragma unroll
      for (int i = LPR / 2; i; i >>= 1) s += __shfl_xor_sync(mask, s, i, LPR);
      const float w = exp2f(s - m);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (w != 0.f) acc[i] = fmaf(w, v[i], acc[i]);
    }
  }
  return make_float4(acc[0], acc[1], acc[2], acc[3]);
}

// VEC: D % 4 == 0 and D <= 128, four dims per lane, LPR lanes per row (D / 4
// rounded up to 16 or 32); else up to 8 strided dims per lane, 32 lanes. Lane i
// takes the (m, l) of part i, so the reads of O wait for nothing but the parts'
// places, and four of them are in flight: with one after the other, a short call of
// 28 parts spent 21 us here; with eight, rows of three or four parts (the usual
// number) execute twice the instructions (256 x 4 x 32 rows: 15 us more). Parts are visited in order, so the sum does not depend
// on which CTA finished first.
template <typename T, int LPR, bool VEC>
__global__ void __launch_bounds__(256)
prefix_join_kernel(const __grid_constant__ PrefixParams p) {
  grid_dependency_wait();
  launch_dependents();
  constexpr int NV = VEC ? 4 : 8;
  // x: token of the batch; y and the CTA's groups of LPR lanes: query heads
  const int lane = threadIdx.x % LPR, D = p.D;
  int hq = blockIdx.y * (blockDim.x / LPR) + threadIdx.x / LPR;
  const bool real = hq < p.H;  // the others follow along for the shuffles
  if (!real) hq = p.H - 1;
  const int bt = blockIdx.x, b = bt / p.T, t = bt - b * p.T, h = hq / p.G, g = hq - h * p.G;
  const int64_t row = (int64_t)bt * p.H + hq;
  int n, count;
  prefix_sequence(p, b, n, count);
  const int limit = prefix_limit(n, count, t);
  PartRange part[2] = {{row, p.rows, 0}, {row, p.rows, 0}};
  if (limit >= 0 && p.prefix.kind) {
    if (p.prefix.kind == kPartSlots)
      part[0].count = p.prefix.slots;
    else
      part[0] = prefix_parts(p.prefix, p.prefix.first + h * p.prefix.segments, bt, g, p.G);
  }
  if (limit > 0) {
    if (p.own.kind == kPartSlots)
      part[1].count = (limit + p.own.chunk - 1) / p.own.chunk;
    else
      part[1] = prefix_parts(p.own, p.own.first + (b * p.KVH + h) * p.own.segments, t, g, p.G);
  }
  const int total = part[0].count + part[1].count;
  // place of part s: its (m, l), and its O
  auto place = [&](int s, const float2** ml) -> const float* {
    const bool first = s < part[0].count;
    const int64_t at = first ? part[0].at + s * part[0].step
                             : part[1].at + (s - part[0].count) * part[1].step;
    *ml = (first ? p.prefix.ml : p.own.ml) + at;
    return (first ? p.prefix.o : p.own.o) + at * D;
  };
  // the same number of rounds for all rows of a warp: the shuffles need every lane
  int rounds = (total + LPR - 1) / LPR;
#pragma unroll
  for (int i = 16; i >= LPR; i >>= 1) rounds = max(rounds, __shfl_xor_sync(0xffffffffu, rounds, i));
  float m = -INFINITY;
  float2 v = make_float2(-INFINITY, 0.f);
  const float* src = nullptr;
  for (int x = 0; x < rounds; ++x) {
    const int s = x * LPR + lane;
    v = make_float2(-INFINITY, 0.f);
    if (s < total) {
      const float2* ml;
      src = place(s, &ml);
      v = *ml;
    }
    m = fmaxf(m, v.x);
  }
#pragma unroll
  for (int i = LPR / 2; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  float l = 0.f, acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  for (int x = 0; x < rounds; ++x) {
    if (rounds > 1) {  // one round: still in registers
      const int s = x * LPR + lane;
      v = make_float2(-INFINITY, 0.f);
      if (s < total) {
        const float2* ml;
        src = place(s, &ml);
        v = *ml;
      }
    }
    const float w = v.x == -INFINITY ? 0.f : exp2f(v.x - m);
    l = fmaf(w, v.y, l);
    const int here = total - x * LPR < LPR ? total - x * LPR : LPR;
    int most = here;
#pragma unroll
    for (int i = 16; i >= LPR; i >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, i));
    auto add = [&](auto width, int s0) {  // parts s0 .. s0 + width - 1
      constexpr int U = decltype(width)::value;
      float ws[U], f[U][NV];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ws[u] = __shfl_sync(0xffffffffu, w, (s0 + u) % LPR, LPR);
        const float* o = reinterpret_cast<const float*>(__shfl_sync(
            0xffffffffu, reinterpret_cast<unsigned long long>(src), (s0 + u) % LPR, LPR));
        const bool in = s0 + u < here;
        if constexpr (VEC) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (in && 4 * lane < D) y = *reinterpret_cast<const float4*>(o + 4 * lane);
          f[u][0] = y.x; f[u][1] = y.y; f[u][2] = y.z; f[u][3] = y.w;
        } else {
#pragma unroll
          for (int i = 0; i < NV; ++i) f[u][i] = in && lane + 32 * i < D ? o[lane + 32 * i] : 0.f;
        }
        if (!in) ws[u] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = fmaf(ws[u], f[u][i], acc[i]);
    };
    constexpr int U = VEC ? 4 : 2;
    for (int s0 = 0; s0 < most; s0 += U) add(std::integral_constant<int, U>{}, s0);
  }
#pragma unroll
  for (int i = LPR / 2; i; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  if constexpr (VEC && sizeof(T) == 2) {
    bool odd = false;  // NaN in the sum alone (a NaN logit is in l too)
#pragma unroll
    for (int i = 0; i < NV; ++i) odd |= acc[i] != acc[i];
    const unsigned mask = LPR == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    if (__ballot_sync(0xffffffffu, odd && real && l == l && l != 0.f) & mask) {
      const float4 y = prefix_row_plain<LPR>(p, row, b, h, limit, m, mask);
      acc[0] = y.x; acc[1] = y.y; acc[2] = y.z; acc[3] = y.w;
    }
  }
  if (!real) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
  T* out = static_cast<T*>(p.out) + (int64_t)row * D;
  if constexpr (VEC) {
    if ((reinterpret_cast<uintptr_t>(p.out) & 15u) == 0) {
      if (4 * lane < D) {
        __align__(16) T o4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o4[i] = Elem<T>::from_f(l == 0.f ? 0.f : acc[i] * inv);
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint2*>(out + 4 * lane) = *reinterpret_cast<const uint2*>(o4);
        else
          *reinterpret_cast<uint4*>(out + 4 * lane) = *reinterpret_cast<const uint4*>(o4);
      }
      if (p.lse && lane == 0) p.lse[row] = l == 0.f ? INFINITY : m + log2f(l);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = VEC ? 4 * lane + i : lane + 32 * i;
    if (d < D) out[d] = Elem<T>::from_f(l == 0.f ? 0.f : acc[i] * inv);
  }
  if (p.lse && lane == 0) p.lse[row] = l == 0.f ? INFINITY : m + log2f(l);
}

// ---- accumulated weights --------------------------------------------------------
// scores_out[b, c, j] = scores[b, c, j] + sum over the T G rows of kv head c that
// see own token j of 2^(logit - lse). Rows are added in order. Four tokens per thread,
// read before any is used: with one each the kernel spent its time in the chain of
// its first reads (16 x 8 heads of 8192 tokens: 15 us against 11).
__global__ void __launch_bounds__(256) prefix_scores_kernel(const PrefixParams p) {
  grid_dependency_wait();
  launch_dependents();
  const int per = (int)((p.scores_width + 1023) / 1024), bh = blockIdx.x / per;
  const int b = bh / p.KVH, h = bh - b * p.KVH;
  const int64_t j0 = (int64_t)(blockIdx.x - bh * per) * 1024 + threadIdx.x;
  const int TG = p.T * p.G;
  constexpr int U = 4;
  const float* in = p.scores + (int64_t)bh * p.scores_width;
  float old[U], add[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t j = j0 + 256 * u;
    old[u] = j < p.scores_width ? in[j] : 0.f;
    add[u] = 0.f;
  }
  int n, count;
  prefix_sequence(p, b, n, count);
  const float* lg = p.logits + (int64_t)bh * p.logits_width * TG;
  if (j0 < n) {
    for (int t = 0; t < count; ++t) {
      const int limit = prefix_limit(n, count, t);
      const float* lse = p.lse + ((int64_t)b * p.T + t) * p.H + (int64_t)h * p.G;
      for (int g = 0; g < p.G; g += 4) {
        float v[U][4], e[4];
        const int here = p.G - g < 4 ? p.G - g : 4;
        const bool wide = (TG & 3) == 0 && here == 4 && (p.G & 3) == 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t j = j0 + 256 * u;
          const float* src = lg + j * TG + t * p.G + g;
          if (wide) {
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j < limit) y = *reinterpret_cast<const float4*>(src);
            v[u][0] = y.x; v[u][1] = y.y; v[u][2] = y.z; v[u][3] = y.w;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = j < limit && i < here ? src[i] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = i < here ? lse[g + i] : INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (j0 + 256 * u < limit)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < here) add[u] += exp2f(v[u][i] - e[i]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t j = j0 + 256 * u;
    if (j < p.scores_width) p.scores_out[(int64_t)bh * p.scores_width + j] = old[u] + add[u];
  }
}

}  // namespace pdb
