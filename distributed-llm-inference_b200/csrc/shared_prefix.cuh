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
//   * the FP32 kernel here: fixed key ranges ("slots") of every row,
//     part index = slot * rows + global row (b T + t) H + h;
//   * the tensor-core kernels: work in units (64- or 128-key tiles of a segment
//     of rows), cut into one contiguous range per CTA; CTA c's piece of segment
//     s is stored as piece s + c (distinct for distinct pieces, as each step to
//     the next piece raises s, c or both), part index = piece * R + row of the
//     segment. The pieces of a segment are those of consecutive CTAs; the first
//     and the last of them are noted in `dir`.
// Either way a row's partials are evenly spaced: prefix_join_kernel joins them.
#pragma once

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

// ---- spans on the FP32 pipes (any type, head_dim <= DP, block size, alignment) --
// One CTA per (row tile of RT, kv head, key range), keys in tiles of KT staged
// in shared memory as FP32. Each thread owns a register tile of S and one of O;
// products and sums are FP32 throughout. Grid: x = the prefix's
// (row tile, range) pairs first, then own (sequence, row tile, chunk) triples;
// y = kv head.
template <int DP, int RT>
struct PrefixSimt {
  static constexpr int NT = 128;
  static constexpr int KT = 32;
  static constexpr int LD = DP + 4;  // padded row of K and Q: rows 4 banks apart
  static constexpr int TPR = NT / RT;        // threads that share a row
  static constexpr int SK = KT / TPR;        // keys per thread of S
  static constexpr int OD = DP / TPR;        // dims per thread of O
  static constexpr size_t SMEM =
      (size_t)(RT * LD + KT * LD + KT * DP + RT * (KT + 1)) * sizeof(float);
};

template <typename T, int DP, int RT>
__global__ void __launch_bounds__(PrefixSimt<DP, RT>::NT)
prefix_simt_kernel(const PrefixParams p, int prefix_tiles, int own_tiles) {
  using C = PrefixSimt<DP, RT>;
  constexpr int NT = C::NT, KT = C::KT, LD = C::LD, TPR = C::TPR, SK = C::SK, OD = C::OD;
  extern __shared__ float smem_f[];
  float* sq = smem_f;            // [RT][LD]
  float* sk = sq + RT * LD;      // [KT][LD]
  float* sv = sk + KT * LD;      // [KT][DP]
  float* sp = sv + KT * DP;      // [RT][KT + 1]
  const int tid = threadIdx.x, h = blockIdx.y, D = p.D, G = p.G;
  grid_dependency_wait();
  launch_dependents();

  // this CTA's rows, keys and slot
  int x = blockIdx.x, b = -1, slot, k0, k1, n = 0, count = 0, width;
  int64_t r0, rend;  // rows of this tile in the kv head's numbering
  const int32_t* table;
  const int npre = prefix_tiles * p.prefix.slots;
  const PartSet& set = x < npre ? p.prefix : p.own;
  if (x < npre) {
    slot = x % set.slots;
    r0 = (int64_t)(x / set.slots) * RT;
    rend = (int64_t)p.B * p.T * G;
    k0 = slot * set.chunk;
    k1 = k0 + set.chunk < p.prefix_length ? k0 + set.chunk : p.prefix_length;
    table = p.prefix_table;
    width = (p.prefix_length + p.block_size - 1) / p.block_size;
  } else {
    x -= npre;
    slot = x % set.slots;
    x /= set.slots;
    const int tile = x % own_tiles;
    b = x / own_tiles;
    prefix_sequence(p, b, n, count);
    r0 = (int64_t)b * p.T * G + (int64_t)tile * RT;
    rend = (int64_t)(b + 1) * p.T * G;
    k0 = slot * set.chunk;
    k1 = k0 + set.chunk < n ? k0 + set.chunk : n;
    table = p.tables + (int64_t)b * p.table_width;
    width = p.table_width;
    if (k0 >= k1) return;
  }
  const T* q = static_cast<const T*>(p.q);
  const T* kp = static_cast<const T*>(p.k_pool);
  const T* vp = static_cast<const T*>(p.v_pool);
  for (int i = tid; i < RT * DP; i += NT) {
    const int r = i / DP, d = i % DP;
    const int64_t row = r0 + r;
    float v = 0.f;
    if (row < rend && d < D)
      v = Elem<T>::to_f(q[((row / G) * p.H + (int64_t)h * G + row % G) * D + d]);
    sq[r * LD + d] = v;
  }
  const int r = tid / TPR, part = tid % TPR;
  const int64_t row = r0 + r;
  int limit = p.prefix_length;  // keys [0, limit) are seen by this thread's row
  if (b >= 0) limit = row < rend ? prefix_limit(n, count, (int)(row / G - (int64_t)b * p.T)) : -1;
  float m = -INFINITY, l = 0.f, acc[OD];
#pragma unroll
  for (int i = 0; i < OD; ++i) acc[i] = 0.f;
  float* logits = (p.logits && b >= 0 && row < rend)
                      ? p.logits + ((int64_t)b * p.KVH + h) * p.logits_width * p.T * G +
                            (row - (int64_t)b * p.T * G)
                      : nullptr;

  for (int t0 = k0; t0 < k1; t0 += KT) {
    __syncthreads();  // the previous tile is consumed
    for (int i = tid; i < KT * DP; i += NT) {
      const int j = i / DP, d = i % DP;
      float kv = 0.f, vv = 0.f;  // keys past the range: zeros, so a zero weight stays zero
      if (t0 + j < k1 && d < D) {
        const int64_t cell = prefix_cell(p, table, width, t0 + j);
        if (cell >= 0) {
          kv = Elem<T>::to_f(kp[(cell * p.KVH + h) * D + d]);
          vv = Elem<T>::to_f(vp[(cell * p.KVH + h) * D + d]);
        }
      }
      sk[j * LD + d] = kv;
      sv[j * DP + d] = vv;
    }
    __syncthreads();
    // S: row r, keys part, part + TPR, ...
    float s[SK];
#pragma unroll
    for (int i = 0; i < SK; ++i) s[i] = 0.f;
    for (int d = 0; d < D; ++d) {
      const float qv = sq[r * LD + d];
#pragma unroll
      for (int i = 0; i < SK; ++i) s[i] = fmaf(qv, sk[(part + i * TPR) * LD + d], s[i]);
    }
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < SK; ++i) {
      const int key = t0 + part + i * TPR;
      s[i] = (key < limit && key < k1) ? s[i] * p.scale_log2 : -INFINITY;
      if (logits && key < limit && key < k1) logits[(int64_t)key * p.T * G] = s[i];
      mt = fmaxf(mt, s[i]);
    }
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
    const float mn = fmaxf(m, mt);
    const float alpha = mn == -INFINITY ? 1.f : exp2f(m - mn);  // m = -inf: 0
#pragma unroll
    for (int i = 0; i < SK; ++i) {
      const float w = s[i] == -INFINITY ? 0.f : exp2f(s[i] - mn);
      l = i == 0 ? l * alpha + w : l + w;
      sp[r * (KT + 1) + part + i * TPR] = w;
    }
    m = mn;
    __syncwarp();  // a row's threads are in one warp
#pragma unroll
    for (int i = 0; i < OD; ++i) acc[i] *= alpha;
    for (int j = 0; j < KT; ++j) {
      const float w = sp[r * (KT + 1) + j];
      if (w == 0.f) continue;  // a key this row does not see: its v may be anything
#pragma unroll
      for (int i = 0; i < OD; ++i) acc[i] = fmaf(w, sv[j * DP + part + i * TPR], acc[i]);
    }
  }
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (row >= rend) return;
  const int64_t at = (int64_t)slot * p.rows + (row / G) * p.H + (int64_t)h * G + row % G;
  if (part == 0) set.ml[at] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < OD; ++i)
    if (part + i * TPR < D) set.o[at * D + part + i * TPR] = acc[i];
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

// VEC: D % 4 == 0 and D <= 128, four dims per lane, LPR lanes per row (D / 4
// rounded up to 16 or 32); else up to 8 strided dims per lane, 32 lanes. Partials
// are visited in order, so the sum does not depend on which CTA finished first.
template <typename T, int LPR, bool VEC>
__global__ void __launch_bounds__(256) prefix_join_kernel(const PrefixParams p) {
  grid_dependency_wait();
  launch_dependents();
  constexpr int NV = VEC ? 4 : 8;
  int row = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR);
  const int lane = threadIdx.x % LPR, D = p.D;
  const bool real = row < p.rows;  // the others follow along for the shuffles
  if (!real) row = (int)p.rows - 1;
  const int bt = row / p.H, b = bt / p.T, t = bt - b * p.T, hq = row - bt * p.H, h = hq / p.G,
            g = hq - h * p.G;
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
  const float2* ml[2] = {p.prefix.ml, p.own.ml};
  const float* o[2] = {p.prefix.o, p.own.o};
  float m = -INFINITY;
#pragma unroll
  for (int x = 0; x < 2; ++x)
    for (int s = lane; s < part[x].count; s += LPR)
      m = fmaxf(m, ml[x][part[x].at + s * part[x].step].x);
#pragma unroll
  for (int i = LPR / 2; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  float l = 0.f, acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll 2
    for (int s = 0; s < part[x].count; ++s) {
      const int64_t at = part[x].at + s * part[x].step;
      const float2 v = ml[x][at];
      const float w = v.x == -INFINITY ? 0.f : exp2f(v.x - m);
      l = fmaf(w, v.y, l);
      if constexpr (VEC) {
        if (4 * lane < D) {
          const float4 f = *reinterpret_cast<const float4*>(o[x] + at * D + 4 * lane);
          acc[0] = fmaf(w, f.x, acc[0]);
          acc[1] = fmaf(w, f.y, acc[1]);
          acc[2] = fmaf(w, f.z, acc[2]);
          acc[3] = fmaf(w, f.w, acc[3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + 32 * i < D) acc[i] = fmaf(w, o[x][at * D + lane + 32 * i], acc[i]);
      }
    }
  }
  if (!real) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
  T* out = static_cast<T*>(p.out) + (int64_t)row * D;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = VEC ? 4 * lane + i : lane + 32 * i;
    if (d < D) out[d] = Elem<T>::from_f(l == 0.f ? 0.f : acc[i] * inv);
  }
  if (p.lse && lane == 0) p.lse[row] = l == 0.f ? INFINITY : m + log2f(l);
}

// ---- accumulated weights --------------------------------------------------------
// scores_out[b, c, j] = scores[b, c, j] + sum over the T G rows of kv head c that
// see own token j of 2^(logit - lse). Rows are added in order.
__global__ void __launch_bounds__(256) prefix_scores_kernel(const PrefixParams p) {
  grid_dependency_wait();
  launch_dependents();
  const int64_t bh = blockIdx.y;
  const int b = (int)(bh / p.KVH), h = (int)(bh % p.KVH);
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j >= p.scores_width) return;
  int n, count;
  prefix_sequence(p, b, n, count);
  float add = 0.f;
  if (j < n) {
    const float* lg = p.logits + (bh * p.logits_width + j) * p.T * p.G;
    for (int t = 0; t < count; ++t) {
      if (j >= prefix_limit(n, count, t)) continue;
      const float* lse = p.lse + ((int64_t)b * p.T + t) * p.H + (int64_t)h * p.G;
      for (int g = 0; g < p.G; ++g) add += exp2f(lg[t * p.G + g] - lse[g]);
    }
  }
  const int64_t at = bh * p.scores_width + j;
  p.scores_out[at] = p.scores[at] + add;
}

}  // namespace pdb
