// Spans of the shared-prefix attention on the warp-level tensor cores, fed by
// TMA (sm_100a, FP16, head_dim 64 / 128, block_size % 16 == 0).
//
// For few rows per key set: a sequence's own tokens (T G rows), or a short
// batch's prefix. Arithmetic intensity is about T G operations per byte, so the
// kernel is bound by HBM and is built to keep reads in flight:
//   * persistent, two CTAs per SM. Segments - (sequence, kv head, row tile) - of
//     ceil(n / 64) key tiles, plus kSpanOverhead units for a segment's start and
//     end, are laid end to end and cut into one contiguous range per CTA of
//     equal length; every CTA derives its range from the device's lengths.
//   * warp 4 is the producer: it walks the range, looks pages up (one lane per
//     16-token unit), and issues one TMA box (16 rows, 64 columns, 128-byte
//     swizzle) per (unit, K|V, column half) into a ring of STAGES tiles; an
//     piece's query rows ride on its first tile's barrier. It runs ahead across
//     piece borders, so the ring never drains between pieces.
//   * warps 0-3 each take 16 SUB keys of a tile and all rows: S^T = K Q^T
//     (keys are the M of the product, so 8 rows cost no more than one), softmax
//     in base 2 with the running maximum raised only when a logit passes it by
//     2^8 (exact after the division; weights stay below 2^8 in FP16), O^T +=
//     V^T P^T with P as a high and a low FP16 term (HILO: the weights keep 22
//     bits; without it 11). At a piece's end the warps' states are joined
//     through the stage just read, 8 rows at a time, and written as its partial.
// Keys past the sequence's end are masked and their V rows zeroed in shared memory.
// A drafted token's V that is not finite must not reach rows that do not see it
// (0 * NaN): such keys are taken out of the product and added row by row.
#pragma once

#include "attention_tma.cuh"
#include "shared_prefix.cuh"

namespace pdb {

// What one launch covers: `nseq` key sets of `rows` rows each; set s belongs to
// tokens s * tokens .. of the batch.
struct SpanSet {
  const int32_t* tables;  // [nseq, width]
  PartSet part;
  int64_t* start;         // [nseq + 1] first unit of each key set, written by CTA 0
  int nseq, width, tokens, rows;
  int own;                // own tokens (lengths, counts, causal) or the prefix
};

struct SpanRec {  // one staged tile, producer -> math warps
  int seq, h, row0, k0, kend, n, count, piece, qbuf, flags, okmask, pad_;
};
constexpr int kSpanFirst = 1, kSpanLast = 2, kSpanEnd = 4;

template <int D_, int NT_, int SUB_, int STAGES_, bool HILO_>
struct SpanMma {
  static constexpr int D = D_, NT = NT_, SUB = SUB_, STAGES = STAGES_;
  static constexpr bool HILO = HILO_;
  static constexpr int ROWS = 8 * NT, TILE = 64 * SUB, UNITS = TILE / 16, HALVES = D / 64;
  static constexpr int KSTEPS = D / 16;
  static constexpr int THREADS = 160;
  static constexpr int TILE_BYTES = TILE * D * 2, STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int QP = D * 2 + 16;  // row pitch of the staged queries (no bank conflicts)
  static constexpr int Q_BYTES = ROWS * QP;
  static constexpr int LCAP = 256;       // lengths and counts kept in shared memory
  static constexpr int JP = D + 4;       // row pitch of the join buffer, in floats
  static_assert(4 * 8 * JP * 4 <= STAGE_BYTES, "join buffer fits a stage");
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + 2 * Q_BYTES +
                                 STAGES * sizeof(SpanRec) + 4 * ROWS * sizeof(float2) +
                                 LCAP * sizeof(int2) + (2 * STAGES + 2) * 8 + 64;
};

constexpr int kSpanOverhead = 1;  // a segment's start and end, in 64-key tiles

template <class C>
__global__ void __launch_bounds__(C::THREADS, 2)
prefix_span_kernel(const PrefixParams p, const SpanSet ss, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  constexpr int D = C::D, NT = C::NT, SUB = C::SUB, STAGES = C::STAGES, TILE = C::TILE;
  constexpr int UNITS = C::UNITS, HALVES = C::HALVES, KSTEPS = C::KSTEPS, ROWS = C::ROWS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto sk = [&](int s) { return base + (size_t)s * C::STAGE_BYTES; };
  auto sv = [&](int s) { return sk(s) + C::TILE_BYTES; };
  unsigned char* sq = base + (size_t)STAGES * C::STAGE_BYTES;  // [2][ROWS][QP]
  float2* mls = reinterpret_cast<float2*>(sq + 2 * C::Q_BYTES);  // [4][ROWS]
  SpanRec* recs = reinterpret_cast<SpanRec*>(mls + 4 * ROWS);    // [STAGES]
  int2* lens = reinterpret_cast<int2*>(recs + STAGES);           // [LCAP]
  uint64_t* full = reinterpret_cast<uint64_t*>(lens + C::LCAP);
  uint64_t* empty = full + STAGES;
  uint64_t* q_empty = empty + STAGES;  // [2]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    mbar_init(&q_empty[0], 4);
    mbar_init(&q_empty[1], 4);
    fence_barrier_init();
  }
  // rows past the item's keep these zeros (their results are never stored)
  for (int i = tid; i < 2 * C::Q_BYTES / 16; i += C::THREADS)
    reinterpret_cast<uint4*>(sq)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  grid_dependency_wait();
  launch_dependents();
  auto length_of = [&](int s) -> int2 {
    int n = p.prefix_length, count = ss.tokens;
    if (ss.own) prefix_sequence(p, s, n, count);
    return make_int2(n, count);
  };
  for (int i = tid; i < ss.nseq && i < C::LCAP; i += C::THREADS) lens[i] = length_of(i);
  __syncthreads();
  bool live = true;  // after one expired wait a thread stops waiting
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (live) live = mbar_wait(bar, parity);
  };

  if (warp == 4) {
    // ---- producer ------------------------------------------------------------
    auto set_length = [&](int s) -> int2 { return s < C::LCAP ? lens[s] : length_of(s); };
    const int64_t per = (int64_t)p.KVH * ss.part.segments;  // segments of a key set
    auto set_units = [&](int s) -> int64_t {
      if (s >= ss.nseq) return 0;
      const int n = set_length(s).x;
      return n > 0 ? per * ((n + 63) / 64 + kSpanOverhead) : 0;
    };
    int64_t total = 0;
    for (int s0 = 0; s0 < ss.nseq; s0 += 32) {
      int64_t w = set_units(s0 + lane);
      if (blockIdx.x == 0 && ss.own) {  // the join needs every sequence's first unit
        int64_t inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        if (s0 + lane < ss.nseq) ss.start[s0 + lane] = total + inc - w;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      total += w;
    }
    if (blockIdx.x == 0 && ss.own && lane == 0) ss.start[ss.nseq] = total;
    const int64_t ctas = unit_ctas(total, gridDim.x);
    const int64_t u0 = blockIdx.x < ctas ? part_begin(blockIdx.x, total, ctas) : total,
                  u1 = blockIdx.x < ctas ? part_begin(blockIdx.x + 1, total, ctas) : total;
    int s = ss.nseq, n = 0, count = 0;
    int64_t u = total, in = 0;  // start of the current segment; its index in the key set
    if (u0 < u1) {
      int64_t run = 0;
      for (int s0 = 0; s0 < ss.nseq; s0 += 32) {
        int64_t inc = set_units(s0 + lane);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const unsigned m = __ballot_sync(0xffffffffu, run + inc > u0);
        if (m) {
          const int f = __ffs(m) - 1;
          s = s0 + f;
          const int64_t before = __shfl_sync(0xffffffffu, inc, f ? f - 1 : 0);
          u = run + (f ? before : 0);
          break;
        }
        run += __shfl_sync(0xffffffffu, inc, 31);
      }
      const int2 nc = set_length(s);
      n = nc.x;
      count = nc.y;
      const int64_t w = (n + 63) / 64 + kSpanOverhead;
      in = (u0 - u) / w;
      u += in * w;
    }
    int64_t g = 0;  // tiles so far
    int item = 0;
    while (u < u1) {
      const int keys = (n + 63) / 64;
      // this CTA's key tiles of the segment: units u + overhead .. are its tiles
      const int64_t lo = u0 - u - kSpanOverhead, hi = u1 - u - kSpanOverhead;
      const int j0 = lo > 0 ? (int)lo : 0, j1 = hi < keys ? (int)hi : keys;
      if (j0 < j1) {
        const int h = (int)(in / ss.part.segments), row0 = (int)(in % ss.part.segments) * ROWS;
        const int nrows = ss.rows - row0 < ROWS ? ss.rows - row0 : ROWS;
        const int k0 = j0 * 64, kend = j1 * 64 < n ? j1 * 64 : n;
        const int qb = item & 1;
        if (item >= 2) wait(&q_empty[qb], (uint32_t)((item >> 1) - 1) & 1u);
        const int32_t* table = ss.tables + (int64_t)s * ss.width;
        for (int t0 = k0; t0 < kend; t0 += TILE, ++g) {
          const int st = (int)(g % STAGES);
          int64_t cell = -1;  // looked up before the wait: the page read hides behind it
          if (lane < UNITS && t0 + lane * 16 < kend)
            cell = prefix_cell(p, table, ss.width, t0 + lane * 16);
          if (g >= STAGES) wait(&empty[st], (uint32_t)(g / STAGES - 1) & 1u);
          const unsigned ok = __ballot_sync(0xffffffffu, cell >= 0);
          const bool first = t0 == k0;
          if (lane == 0) {
            SpanRec r;
            r.seq = s; r.h = h; r.row0 = row0; r.k0 = t0; r.kend = kend; r.n = n; r.count = count;
            r.piece = (int)(s * per + in + blockIdx.x); r.qbuf = qb; r.okmask = (int)ok;
            r.flags = (first ? kSpanFirst : 0) | (t0 + TILE >= kend ? kSpanLast : 0);
            r.pad_ = 0;
            recs[st] = r;
            mbar_arrive_expect_tx(&full[st], (uint32_t)__popc(ok) * 2u * HALVES * 2048u +
                                                 (first ? (uint32_t)nrows * D * 2u : 0u));
          }
          __syncwarp();
          if (first) {
            for (int r = lane; r < nrows; r += 32) {
              const int row = row0 + r;
              const __half* src = static_cast<const __half*>(p.q) +
                                  (((int64_t)s * ss.tokens + row / p.G) * p.H + (int64_t)h * p.G +
                                   row % p.G) * D;
              bulk_load(sq + qb * C::Q_BYTES + r * C::QP, src, D * 2, &full[st]);
            }
          }
          if (cell >= 0) {
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf) {
              const int dst = hf * (TILE * 128) + lane * 2048;
              tma_load_3d(sk(st) + dst, &kmap, hf * 64, h, (int)cell, &full[st]);
              tma_load_3d(sv(st) + dst, &vmap, hf * 64, h, (int)cell, &full[st]);
            }
          }
        }
        ++item;
      }
      u += keys + kSpanOverhead;
      if (++in == per) {  // next key set that holds keys
        in = 0;
        n = 0;
        while (n <= 0 && ++s < ss.nseq) {
          const int2 nc = set_length(s);
          n = nc.x;
          count = nc.y;
        }
        if (n <= 0) break;
      }
    }
    const int st = (int)(g % STAGES);
    if (g >= STAGES) wait(&empty[st], (uint32_t)(g / STAGES - 1) & 1u);
    if (lane == 0) {
      recs[st].flags = kSpanEnd;
      mbar_arrive(&full[st]);
    }
    return;
  }

  // ---- math warps --------------------------------------------------------------
  const int gq = lane >> 2, tg = lane & 3, mi = lane >> 3;
  auto offset = [](int row, int col) {  // 16-byte chunk `col` of staged row `row`
    return (col >> 3) * (TILE * 128) + row * 128 + (((col & 7) ^ (row & 7)) << 4);
  };
  float m[NT][2], l[NT][2], acc[KSTEPS][NT][4];
  for (int64_t g = 0;; ++g) {
    const int st = (int)(g % STAGES);
    wait(&full[st], (uint32_t)(g / STAGES) & 1u);
    const SpanRec r = recs[st];
    if (r.flags & kSpanEnd || !live) break;
    if (r.flags & kSpanFirst) {
#pragma unroll
      for (int i = 0; i < NT; ++i) m[i][0] = m[i][1] = -INFINITY, l[i][0] = l[i][1] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[k][i][e] = 0.f;
    }
    const int w0 = warp * 16 * SUB;  // this warp's first key of the tile
    const int left = r.kend - r.k0 - w0;
    if (left > 0) {
      unsigned char* k_s = sk(st);
      unsigned char* v_s = sv(st);
      // rows past the end: zero V; units without a page: zero K and V
      bool wrote = false;
#pragma unroll
      for (int sb = 0; sb < SUB; ++sb) {
        const int unit = warp * SUB + sb;
        const bool bad = left > 16 * sb && !(r.okmask >> unit & 1);
        const int keep = bad ? 0 : (left - 16 * sb < 0 ? 0 : left - 16 * sb);
        if (keep < 16) {
          wrote = true;
          for (int i = lane; i < (16 - keep) * (D / 8); i += 32) {
            const int row = w0 + 16 * sb + keep + i / (D / 8);
            *reinterpret_cast<uint4*>(v_s + offset(row, i % (D / 8))) = make_uint4(0, 0, 0, 0);
            if (bad) *reinterpret_cast<uint4*>(k_s + offset(row, i % (D / 8))) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      if (wrote) __syncwarp();

      float sc[SUB][NT][4];  // [key gq | gq + 8] x [row 2 tg | 2 tg + 1]
#pragma unroll
      for (int sb = 0; sb < SUB; ++sb)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[sb][i][e] = 0.f;
      const unsigned char* q_s = sq + r.qbuf * C::Q_BYTES + (lane & 7) * C::QP;
#pragma unroll
      for (int k2 = 0; k2 < KSTEPS / 2; ++k2) {
        uint32_t qb[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
          ldsm_x4(qb[i][0], qb[i][1], qb[i][2], qb[i][3], q_s + i * 8 * C::QP + (4 * k2 + mi) * 16);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
          for (int sb = 0; sb < SUB; ++sb) {
            uint32_t a0, a1, a2, a3;
            const int row = w0 + 16 * sb + ((mi & 1) << 3) + (lane & 7);
            ldsm_x4(a0, a1, a2, a3, k_s + offset(row, 2 * (2 * k2 + kk) + (mi >> 1)));
#pragma unroll
            for (int i = 0; i < NT; ++i)
              mma_16816(sc[sb][i], a0, a1, a2, a3, qb[i][2 * kk], qb[i][2 * kk + 1]);
          }
        }
      }
      // scale, mask, store logits
      const int key0 = r.k0 + w0 + gq;
      const bool causal = ss.own && r.count > 1 && r.k0 + w0 + 16 * SUB > r.n - r.count + 1;
      const bool edge = left < 16 * SUB || causal;
#pragma unroll
      for (int sb = 0; sb < SUB; ++sb)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = sc[sb][i][e] * p.scale_log2;
            if (edge) {
              const int key = key0 + 16 * sb + (e >> 1) * 8;
              int lim = r.kend;
              if (causal) {
                const int own_lim = prefix_limit(r.n, r.count, (r.row0 + 8 * i + 2 * tg + (e & 1)) / p.G);
                lim = own_lim < lim ? own_lim : lim;
              }
              if (key >= lim) x = -INFINITY;
            }
            sc[sb][i][e] = x;
          }
      if (p.logits && ss.own) {
        float* lg = p.logits + ((int64_t)r.seq * p.KVH + r.h) * p.logits_width * ss.rows;
#pragma unroll
        for (int sb = 0; sb < SUB; ++sb)
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const int key = key0 + 16 * sb + 8 * e2;
            if (key < r.kend) {
              float* at = lg + (int64_t)key * ss.rows + r.row0 + 2 * tg;
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                const int row = r.row0 + 8 * i + 2 * tg;
                if (ss.rows % 2 == 0) {
                  if (row < ss.rows)
                    *reinterpret_cast<float2*>(at + 8 * i) =
                        make_float2(sc[sb][i][2 * e2], sc[sb][i][2 * e2 + 1]);
                } else {
                  if (row < ss.rows) at[8 * i] = sc[sb][i][2 * e2];
                  if (row + 1 < ss.rows) at[8 * i + 1] = sc[sb][i][2 * e2 + 1];
                }
              }
            }
          }
      }
      // running maxima
      float mx[NT][2];
      bool grow = false;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[0][i][e], sc[0][i][e + 2]);
#pragma unroll
          for (int sb = 1; sb < SUB; ++sb) x = fmaxf(x, fmaxf(sc[sb][i][e], sc[sb][i][e + 2]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          mx[i][e] = x;
          grow |= x > m[i][e] + 8.f;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float nm = fmaxf(m[i][e], mx[i][e]);
            const float a = nm == -INFINITY ? 1.f : exp2f(m[i][e] - nm);
            m[i][e] = nm;
            l[i][e] *= a;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
              acc[k][i][e] *= a;
              acc[k][i][e + 2] *= a;
            }
          }
      }
      uint32_t bh[SUB][NT][2], bl[SUB][NT][2];
#pragma unroll
      for (int sb = 0; sb < SUB; ++sb)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = sc[sb][i][e];
            w[e] = x == -INFINITY ? 0.f : exp2f(x - m[i][e & 1]);
            l[i][e & 1] += w[e];
            sc[sb][i][e] = w[e];
          }
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const uint32_t hi = pack_half2(w[2 * e2], w[2 * e2 + 1]);
            bh[sb][i][e2] = movmatrix_t(hi);
            if constexpr (C::HILO) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              bl[sb][i][e2] = movmatrix_t(pack_half2(w[2 * e2] - f.x, w[2 * e2 + 1] - f.y));
            }
          }
        }
      if (causal) {
        // keys of this warp that some row must not see: their V has to be finite
        const int from = r.n - r.count + 1 - (r.k0 + w0);
        for (int j = from < 0 ? 0 : from; j < 16 * SUB && j < left; ++j) {
          bool odd = false;
          for (int cc = lane; cc < D / 8; cc += 32) {
            const uint4 x = *reinterpret_cast<const uint4*>(v_s + offset(w0 + j, cc));
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              odd |= (words[e] & 0x7c00u) == 0x7c00u || (words[e] & 0x7c000000u) == 0x7c000000u;
          }
          if (!__any_sync(0xffffffffu, odd)) continue;
          wrote = true;
          const int src = (j & 7) * 4 + tg;  // the lane that holds key j's weights of these rows
#pragma unroll
          for (int sb = 0; sb < SUB; ++sb)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const float lo0 = __shfl_sync(0xffffffffu, sc[sb][i][0], src);
              const float lo1 = __shfl_sync(0xffffffffu, sc[sb][i][1], src);
              const float hi0 = __shfl_sync(0xffffffffu, sc[sb][i][2], src);
              const float hi1 = __shfl_sync(0xffffffffu, sc[sb][i][3], src);
              if ((j >> 4) != sb) continue;
              const float w0r = j & 8 ? hi0 : lo0, w1r = j & 8 ? hi1 : lo1;
#pragma unroll
              for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                  const int d = 16 * k + gq + 8 * e2;
                  const float x = __half2float(*reinterpret_cast<const __half*>(
                      v_s + offset(w0 + j, d >> 3) + (d & 7) * 2));
                  if (w0r != 0.f) acc[k][i][2 * e2] += w0r * x;
                  if (w1r != 0.f) acc[k][i][2 * e2 + 1] += w1r * x;
                }
            }
          __syncwarp();
          for (int cc = lane; cc < D / 8; cc += 32)
            *reinterpret_cast<uint4*>(v_s + offset(w0 + j, cc)) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int sb = 0; sb < SUB; ++sb) {
        const int vrow = w0 + 16 * sb + ((mi >> 1) << 3) + (lane & 7);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          uint32_t a0, a1, a2, a3;
          ldsm_x4_t(a0, a1, a2, a3, v_s + offset(vrow, 2 * k + (mi & 1)));
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            mma_16816(acc[k][i], a0, a1, a2, a3, bh[sb][i][0], bh[sb][i][1]);
            if constexpr (C::HILO)
              mma_16816(acc[k][i], a0, a1, a2, a3, bl[sb][i][0], bl[sb][i][1]);
          }
        }
      }
      if (wrote) fence_proxy_async_smem();  // before the next TMA write of this stage
    }
    if (r.flags & kSpanLast) {
      // join of the four warps' states through this stage, 8 rows at a time
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[i][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
          if (gq == 0) mls[warp * ROWS + 8 * i + 2 * tg + e] = make_float2(m[i][e], x);
        }
      named_bar_sync(1, 128);  // states published; every warp is done with the stage
      if (lane == 0) mbar_arrive(&q_empty[r.qbuf]);
      float* jb = reinterpret_cast<float*>(sk(st));  // [4][8][JP]
      const int jr = tid >> 4, part = tid & 15;      // row and 1/16 of its dims
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (r.row0 + 8 * i >= ss.rows) break;  // CTA-uniform
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * i + 2 * tg + e;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < 4; ++w) top = fmaxf(top, mls[w * ROWS + row].x);
          const float a = m[i][e] == -INFINITY ? 0.f : exp2f(m[i][e] - top);
          float* dst = jb + (warp * 8 + 2 * tg + e) * C::JP + gq;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            // a = 0: this warp saw no key of the row; acc is 0 then
            dst[16 * k] = acc[k][i][e] * a;
            dst[16 * k + 8] = acc[k][i][e + 2] * a;
          }
        }
        named_bar_sync(1, 128);
        const int row = r.row0 + 8 * i + jr;
        if (row < ss.rows) {
          const int64_t at = (int64_t)r.piece * ROWS + 8 * i + jr;
          float* og = ss.part.o + at * D;
#pragma unroll
          for (int q4 = 0; q4 < D / 64; ++q4) {
            const int d = (q4 * 16 + part) * 4;
            float4 sum = *reinterpret_cast<const float4*>(jb + jr * C::JP + d);
#pragma unroll
            for (int w = 1; w < 4; ++w) {
              const float4 x = *reinterpret_cast<const float4*>(jb + (w * 8 + jr) * C::JP + d);
              sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
            }
            *reinterpret_cast<float4*>(og + d) = sum;
          }
          if (part == 0) {
            float top = -INFINITY, ls = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, mls[w * ROWS + 8 * i + jr].x);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float2 x = mls[w * ROWS + 8 * i + jr];
              ls += x.y * (x.x == -INFINITY ? 0.f : exp2f(x.x - top));  // a NaN sum stays NaN
            }
            ss.part.ml[at] = make_float2(top, ls);
          }
        }
        named_bar_sync(1, 128);  // the buffer (and, last, the states) may be rewritten
      }
      fence_proxy_async_smem();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
  }
}

}  // namespace pdb
