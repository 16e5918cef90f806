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
//     16-token unit), and issues one TMA box (64 columns, 16 rows, all column
//     halves of one head; 128-byte swizzle) per (unit, K|V) into a ring of STAGES
//     tiles. A box costs the TMA unit about 48 cycles plus 0.9 per row of 128
//     bytes (measured: 2 KB boxes 34 bytes a cycle, 4 KB 53, 16 KB 107), so one box
//     takes both halves. An
//     piece's query rows ride on its first tile's barrier. It runs ahead across
//     piece borders, so the ring never drains between pieces.
//   * warps 0-3: each takes 16 KB keys of a tile and 8 NT rows; with more than 16
//     rows two warps share the keys and split the rows (RW = 2), as all of them
//     in one warp's registers would spill (measured: 7400 cycles a tile instead of
//     2700 at 32 rows). S^T = K Q^T (keys are the M of the product, so 8 rows
//     cost no more than one), softmax in base 2 with the running maximum raised
//     only when a logit passes it by 2^8 (exact after the division; weights stay
//     below 2^8 in FP16), O^T += V^T P^T. P is two FP16 terms, its rounding and the
//     rounded rest (22 bits): one alone is off by 2^-11 of each weight, as much as
//     rounding the output adds. At a piece's end the warps' states are joined through
//     the stage just read, 8 RW rows at a time, and written as its partial.
// Keys that do not count (past the end, or without a page) are masked in the
// logits and in the V fragments, so what their staged rows hold does not matter.
// A drafted token's V that is not finite must not reach rows that do not see it
// (0 * NaN): such keys are masked alike and added row by row.
#pragma once

#include "prefill_tc.cuh"
#include "shared_prefix.cuh"

namespace pdb {

// What one launch covers: key sets of B own contexts (rows T G each) and, before
// them, the prefix (rows B T G) when it has few rows. Segments are numbered through
// both: the prefix's first, then those of sequence 0, 1, ..
struct SpanSet {
  PartSet part;               // segments: per own context and kv head
  int has_prefix, nseq;       // key sets: has_prefix + nseq
  int prefix_segments;        // per kv head
  int beside;                 // the previous kernel in the stream is this call's prefix kernel, whose
                              // CTAs let this one start only once all work before it was complete:
                              // nothing here waits for it but the end
};

struct SpanRec {  // one staged tile, producer -> math warps
  int seq;  // sequence, or -1: the prefix
  int h, row0, rows, k0, kend, n, count, piece, qbuf, flags, okmask;
};
constexpr int kSpanFirst = 1, kSpanLast = 2, kSpanEnd = 4;

template <int D_, int NT_, int RW_, int STAGES_>
struct SpanMma {
  static constexpr int D = D_, NT = NT_, RW = RW_, STAGES = STAGES_;
  static constexpr int ROWS = 8 * NT * RW, TILE = D == 64 ? 128 : 64, UNITS = TILE / 16;
  static constexpr int KW = 4 / RW;           // warps that split a tile's keys
  static constexpr int KB = UNITS / KW;       // 16-key blocks per warp
  static constexpr int KSTEPS = D / 16;
  static constexpr int THREADS = 160;
  static constexpr int UNIT_BYTES = 16 * D * 2;  // [D / 64][16 rows][128 bytes], as one box leaves it
  static constexpr int TILE_BYTES = TILE * D * 2, STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int QP = D * 2 + 16;  // row pitch of the staged queries (no bank conflicts)
  static constexpr int Q_BYTES = ROWS * QP;
  static constexpr int LCAP = 256;       // lengths and counts kept in shared memory
  static constexpr int JP = D + 4;       // row pitch of the join buffer, in floats
  static_assert(4 * 8 * JP * 4 <= STAGE_BYTES, "join buffer fits a stage");
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + 2 * Q_BYTES +
                                 STAGES * sizeof(SpanRec) + KW * ROWS * sizeof(float2) +
                                 LCAP * sizeof(int2) + (2 * STAGES + 2) * 8 + 64;
};

constexpr int kSpanOverhead = 1;  // a segment's start and end, in 64-key tiles

__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z,
                                            int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, 2)
prefix_span_kernel(const PrefixParams p, const SpanSet ss, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  constexpr int D = C::D, NT = C::NT, KB = C::KB, KW = C::KW, STAGES = C::STAGES, TILE = C::TILE;
  constexpr int UNITS = C::UNITS, KSTEPS = C::KSTEPS, ROWS = C::ROWS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto sk = [&](int s) { return base + (size_t)s * C::STAGE_BYTES; };
  auto sv = [&](int s) { return sk(s) + C::TILE_BYTES; };
  unsigned char* sq = base + (size_t)STAGES * C::STAGE_BYTES;  // [2][ROWS][QP]
  float2* mls = reinterpret_cast<float2*>(sq + 2 * C::Q_BYTES);  // [KW][ROWS]
  SpanRec* recs = reinterpret_cast<SpanRec*>(mls + KW * ROWS);    // [STAGES]
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
  if (tid == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (!ss.beside) grid_dependency_wait();
  launch_dependents();
  const int sets = ss.has_prefix + ss.nseq;
  auto length_of = [&](int s) -> int2 {  // keys and tokens of key set s
    int n = p.prefix_length, count = p.B * p.T;
    if (s >= ss.has_prefix) prefix_sequence(p, s - ss.has_prefix, n, count);
    return make_int2(n, count);
  };
  for (int i = tid; i < sets && i < C::LCAP; i += C::THREADS) lens[i] = length_of(i);
  __syncthreads();
  bool live = true;  // after one expired wait a thread stops waiting
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (live) live = mbar_wait(bar, parity);
  };

  if (warp == 4) {
    // ---- producer ------------------------------------------------------------
    auto set_length = [&](int s) -> int2 { return s < C::LCAP ? lens[s] : length_of(s); };
    // segments of a key set, and of those before it
    const int own_per = p.KVH * ss.part.segments, prefix_per = p.KVH * ss.prefix_segments;
    auto per = [&](int s) { return s < ss.has_prefix ? prefix_per : own_per; };
    auto set_units = [&](int s) -> int {
      if (s >= sets) return 0;
      const int n = set_length(s).x;
      return n > 0 ? per(s) * ((n + 63) / 64 + kSpanOverhead) : 0;
    };
    int total = 0;
    for (int s0 = 0; s0 < sets; s0 += 32)
      total += (int)__reduce_add_sync(0xffffffffu, (unsigned)set_units(s0 + lane));
    const int ctas = unit_ctas(total, (int)gridDim.x), me = (int)blockIdx.x;
    const int u0 = unit_begin(me, total, ctas), u1 = unit_begin(me + 1, total, ctas);
    int s = sets, n = 0, count = 0;
    int u = total, in = 0;  // start of the current segment; its index in the key set
    if (u0 < u1) {
      int run = 0;
      for (int s0 = 0; s0 < sets; s0 += 32) {
        const int w = set_units(s0 + lane);
        int inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const unsigned m = __ballot_sync(0xffffffffu, run + inc > u0);
        if (m) {
          const int f = __ffs(m) - 1;
          s = s0 + f;
          u = run + __shfl_sync(0xffffffffu, inc - w, f);
          break;
        }
        run += __shfl_sync(0xffffffffu, inc, 31);
      }
      const int2 nc = set_length(s);
      n = nc.x;
      count = nc.y;
      const int w = (n + 63) / 64 + kSpanOverhead;
      in = (u0 - u) / w;
      u += in * w;
    }
    int g = 0;  // tiles so far
    int item = 0;
    while (u < u1) {
      const int keys = (n + 63) / 64;
      // this CTA's key tiles of the segment: units u + overhead .. are its tiles
      const int lo = u0 - u - kSpanOverhead, hi = u1 - u - kSpanOverhead;
      const int j0 = lo > 0 ? lo : 0, j1 = hi < keys ? hi : keys;
      if (j0 < j1) {
        const bool own = s >= ss.has_prefix;
        const int seq = own ? s - ss.has_prefix : -1;
        const int seg = (own ? ss.has_prefix * prefix_per + seq * own_per : 0) + in;
        const int segments = own ? ss.part.segments : ss.prefix_segments;
        const int token0 = own ? seq * p.T : 0, rows = (own ? p.T : p.B * p.T) * p.G;
        const int32_t* table = own ? p.tables + (int64_t)seq * p.table_width : p.prefix_table;
        const int width = own ? p.table_width : (p.prefix_length + p.block_size - 1) / p.block_size;
        if (lane == 0 && j0 == 0) ss.part.dir[seg].x = me;
        if (lane == 0 && j1 == keys) ss.part.dir[seg].y = me;
        const int h = in / segments, row0 = (in - h * segments) * ROWS;
        const int nrows = rows - row0 < ROWS ? rows - row0 : ROWS;
        const int k0 = j0 * 64, kend = j1 * 64 < n ? j1 * 64 : n;
        const int qb = item & 1;
        if (item >= 2) wait(&q_empty[qb], (uint32_t)((item >> 1) - 1) & 1u);
        for (int t0 = k0; t0 < kend; t0 += TILE, ++g) {
          const int st = (int)(g % STAGES);
          int64_t cell = -1;  // looked up before the wait: the page read hides behind it
          if (lane < UNITS && t0 + lane * 16 < kend)
            cell = prefix_cell(p, table, width, t0 + lane * 16);
          if (g >= STAGES) wait(&empty[st], (uint32_t)(g / STAGES - 1) & 1u);
          const unsigned ok = __ballot_sync(0xffffffffu, cell >= 0);
          const bool first = t0 == k0;
          if (lane == 0) {
            SpanRec r;
            r.seq = seq; r.h = h; r.row0 = row0; r.rows = rows; r.k0 = t0; r.kend = kend; r.n = n; r.count = count;
            r.piece = seg + me; r.qbuf = qb; r.okmask = (int)ok;
            r.flags = (first ? kSpanFirst : 0) | (t0 + TILE >= kend ? kSpanLast : 0);
            recs[st] = r;
            mbar_arrive_expect_tx(&full[st], (uint32_t)__popc(ok) * 2u * C::UNIT_BYTES +
                                                 (first ? (uint32_t)nrows * D * 2u : 0u));
          }
          __syncwarp();
          if (first) {
            for (int r = lane; r < nrows; r += 32) {
              const int row = row0 + r;
              const __half* src = static_cast<const __half*>(p.q) +
                                  ((int64_t)(token0 + row / p.G) * p.H + (int64_t)h * p.G +
                                   row % p.G) * D;
              bulk_load(sq + qb * C::Q_BYTES + r * C::QP, src, D * 2, &full[st]);
            }
          }
          int from[UNITS];
#pragma unroll
          for (int i = 0; i < UNITS; ++i) from[i] = __shfl_sync(0xffffffffu, (int)cell, i);
          if (lane == 0) {
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
              if (from[i] < 0) continue;
              tma_load_4d(sk(st) + i * C::UNIT_BYTES, &kmap, 0, from[i], 0, h, &full[st]);
              tma_load_4d(sv(st) + i * C::UNIT_BYTES, &vmap, 0, from[i], 0, h, &full[st]);
            }
          }
          __syncwarp();
        }
        ++item;
      }
      u += keys + kSpanOverhead;
      if (++in == per(s)) {  // next key set that holds keys
        in = 0;
        n = 0;
        while (n <= 0 && ++s < sets) {
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
    if (ss.beside) grid_dependency_wait();  // the join that follows needs the prefix kernel too
    return;
  }

  // ---- math warps --------------------------------------------------------------
  const int gq = lane >> 2, tg = lane & 3, mi = lane >> 3;
  const int kw = warp % KW, rw = warp / KW;  // this warp's keys and rows
  const int rows0 = rw * 8 * NT;
  // Staged row `row` (of 16) of a unit, 16-byte chunk `col`: the swizzle XORs the
  // chunk with row & 7. Per lane: rows and chunks that its ldmatrix addresses name.
  const int krow = ((mi & 1) << 3) + (lane & 7), vrow = ((mi >> 1) << 3) + (lane & 7);
  const int klane = kw * KB * C::UNIT_BYTES + krow * 128 + (((mi >> 1) ^ (krow & 7)) << 4);
  const int vlane = kw * KB * C::UNIT_BYTES + vrow * 128 + (((mi & 1) ^ (vrow & 7)) << 4);
  const int qlane = (rows0 + (lane & 7)) * C::QP + mi * 16;
  float m[NT][2], l[NT][2], acc[KSTEPS][NT][4];
  // Round -1 runs the tile's code on whatever the first stage holds, while the
  // first tile is on its way, and throws the result away: what it brings is the
  // code itself, whose first execution otherwise waits on instruction fetches
  // (1 to 3 us of calls that take 15 to 40).
  for (int g = -1;; ++g) {
    const int st = g < 0 ? 0 : g % STAGES;
    SpanRec r;
    if (g >= 0) {
      wait(&full[st], (uint32_t)(g / STAGES) & 1u);
      r = recs[st];
      if (r.flags & kSpanEnd || !live) break;
    } else {
      r.seq = r.h = r.row0 = r.rows = r.k0 = r.piece = r.qbuf = r.count = 0;
      r.kend = r.n = TILE;
      r.flags = kSpanFirst;
      r.okmask = -1;
    }
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
    const int w0 = kw * 16 * KB;           // this warp's first key of the tile
    const int left = r.kend - r.k0 - w0;   // its keys that count
    if (left > 0) {
      const unsigned char* v_s = sv(st);
      float sc[KB][NT][4];  // [key gq | gq + 8] x [row 2 tg | 2 tg + 1]
#pragma unroll
      for (int sb = 0; sb < KB; ++sb)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[sb][i][e] = 0.f;
      {
        const unsigned char* q_s = sq + r.qbuf * C::Q_BYTES + qlane;
        const unsigned char* k_s = sk(st) + klane;
        const int kx = klane & 0x70;  // chunk bits of the lane's address
#pragma unroll
        for (int k2 = 0; k2 < KSTEPS / 2; ++k2) {
          uint32_t qb[NT][4];
#pragma unroll
          for (int i = 0; i < NT; ++i)
            ldsm_x4(qb[i][0], qb[i][1], qb[i][2], qb[i][3], q_s + i * 8 * C::QP + k2 * 64);
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            const int ks = 2 * k2 + kk;
            const int at = (ks >> 2) * 2048 - kx + (kx ^ ((ks & 3) << 5));
#pragma unroll
            for (int sb = 0; sb < KB; ++sb) {
              uint32_t a0, a1, a2, a3;
              ldsm_x4(a0, a1, a2, a3, k_s + sb * C::UNIT_BYTES + at);
#pragma unroll
              for (int i = 0; i < NT; ++i)
                mma_16816(sc[sb][i], a0, a1, a2, a3, qb[i][2 * kk], qb[i][2 * kk + 1]);
            }
          }
        }
      }
      // scale, mask
      const int key0 = r.k0 + w0 + gq;
      const bool causal = r.seq >= 0 && r.count > 1 && r.k0 + w0 + 16 * KB > r.n - r.count + 1;
      const unsigned units = (unsigned)r.okmask >> (kw * KB);
      const bool edge = left < 16 * KB || causal || (units & ((1u << KB) - 1)) != (1u << KB) - 1;
      // V fragments: keys 2 tg, 2 tg + 1 (low, high half) and those 8 on
      uint32_t keep[KB][2];
#pragma unroll
      for (int sb = 0; sb < KB; ++sb) keep[sb][0] = keep[sb][1] = 0xffffffffu;
#pragma unroll
      for (int sb = 0; sb < KB; ++sb)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[sb][i][e] *= p.scale_log2;
      if (edge) {
        int lim[NT][2];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            lim[i][e] = r.kend;
            if (causal) {
              const int own = prefix_limit(r.n, r.count, (r.row0 + rows0 + 8 * i + 2 * tg + e) / p.G);
              lim[i][e] = own < lim[i][e] ? own : lim[i][e];
            }
          }
#pragma unroll
        for (int sb = 0; sb < KB; ++sb) {
          const bool ok = units >> sb & 1;
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (!ok) sc[sb][i][e] = 0.f;  // no page: reads as zeros
              if (key0 + 16 * sb + (e >> 1) * 8 >= lim[i][e & 1]) sc[sb][i][e] = -INFINITY;
            }
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const int j = 16 * sb + 2 * tg + 8 * e2;
            if (!ok || j >= left) keep[sb][e2] &= 0xffff0000u;
            if (!ok || j + 1 >= left) keep[sb][e2] &= 0x0000ffffu;
          }
        }
      }
      if (p.logits && r.seq >= 0 && g >= 0) {
        float* lg = p.logits + ((int64_t)r.seq * p.KVH + r.h) * p.logits_width * r.rows;
#pragma unroll
        for (int sb = 0; sb < KB; ++sb)
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const int key = key0 + 16 * sb + 8 * e2;
            if (key < r.kend) {
#pragma unroll
              for (int i = 0; i < NT; ++i) {
                const int row = r.row0 + rows0 + 8 * i + 2 * tg;
                float* at = lg + (int64_t)key * r.rows + row;
                if (r.rows % 2 == 0) {
                  if (row < r.rows)
                    *reinterpret_cast<float2*>(at) =
                        make_float2(sc[sb][i][2 * e2], sc[sb][i][2 * e2 + 1]);
                } else {
                  if (row < r.rows) at[0] = sc[sb][i][2 * e2];
                  if (row + 1 < r.rows) at[1] = sc[sb][i][2 * e2 + 1];
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
          for (int sb = 1; sb < KB; ++sb) x = fmax3(x, sc[sb][i][e], sc[sb][i][e + 2]);
          mx[i][e] = x;
        }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            mx[i][e] = fmaxf(mx[i][e], __shfl_xor_sync(0xffffffffu, mx[i][e], o));
#pragma unroll
      for (int i = 0; i < NT; ++i) grow |= mx[i][0] > m[i][0] + 8.f || mx[i][1] > m[i][1] + 8.f;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float nm = fmaxf(m[i][e], mx[i][e]);
            const float a = nm == -INFINITY ? 1.f : ex2(m[i][e] - nm);
            m[i][e] = nm;
            l[i][e] *= a;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
              acc[k][i][e] *= a;
              acc[k][i][e + 2] *= a;
            }
          }
      }
      uint32_t bh[KB][NT][2], bl[KB][NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        // a row without a logit yet: any finite reference gives weights 0
        const float ref0 = m[i][0] == -INFINITY ? 0.f : m[i][0];
        const float ref1 = m[i][1] == -INFINITY ? 0.f : m[i][1];
#pragma unroll
        for (int sb = 0; sb < KB; ++sb)
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const float w0r = ex2(sc[sb][i][2 * e2] - ref0), w1r = ex2(sc[sb][i][2 * e2 + 1] - ref1);
            l[i][0] += w0r;
            l[i][1] += w1r;
            sc[sb][i][2 * e2] = w0r;
            sc[sb][i][2 * e2 + 1] = w1r;
            const uint32_t hi = pack_half2(w0r, w1r);
            bh[sb][i][e2] = movmatrix_t(hi);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            bl[sb][i][e2] = movmatrix_t(pack_half2(w0r - f.x, w1r - f.y));
          }
      }
      if (causal) {
        // keys that some row must not see: their V has to be finite in the product
        const int from = r.n - r.count + 1 - (r.k0 + w0);
        for (int j = from < 0 ? 0 : from; j < 16 * KB && j < left; ++j) {
          const unsigned char* vr = v_s + (kw * KB + (j >> 4)) * C::UNIT_BYTES + (j & 15) * 128;
          bool odd = false;
          if (lane < D / 8) {
            const uint4 x = *reinterpret_cast<const uint4*>(vr + (lane >> 3) * 2048 + (lane & 7) * 16);
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              odd |= (words[e] & 0x7c00u) == 0x7c00u || (words[e] & 0x7c000000u) == 0x7c000000u;
          }
          if (!__any_sync(0xffffffffu, odd)) continue;
          const int src = (j & 7) * 4 + tg;  // the lane that holds key j's weights of these rows
#pragma unroll
          for (int sb = 0; sb < KB; ++sb) {
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
                      vr + (d >> 6) * 2048 + ((((d >> 3) & 7) ^ (j & 7)) << 4) + (d & 7) * 2));
                  if (w0r != 0.f) acc[k][i][2 * e2] += w0r * x;
                  if (w1r != 0.f) acc[k][i][2 * e2 + 1] += w1r * x;
                }
            }
            if ((j >> 4) == sb && ((j & 7) >> 1) == tg) {
              const uint32_t mask = j & 1 ? 0x0000ffffu : 0xffff0000u;
              if (j & 8) keep[sb][1] &= mask;
              else keep[sb][0] &= mask;
            }
          }
        }
      }
      // O^T += V^T P^T
      {
        const unsigned char* v_l = v_s + vlane;
        const int vx = vlane & 0x70;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const int at = (k >> 2) * 2048 - vx + (vx ^ ((k & 3) << 5));
#pragma unroll
          for (int sb = 0; sb < KB; ++sb) {
            uint32_t a0, a1, a2, a3;
            ldsm_x4_t(a0, a1, a2, a3, v_l + sb * C::UNIT_BYTES + at);
            a0 &= keep[sb][0];
            a1 &= keep[sb][0];
            a2 &= keep[sb][1];
            a3 &= keep[sb][1];
#pragma unroll
            for (int i = 0; i < NT; ++i)
              mma_16816(acc[k][i], a0, a1, a2, a3, bh[sb][i][0], bh[sb][i][1]);
#pragma unroll
            for (int i = 0; i < NT; ++i)
              mma_16816(acc[k][i], a0, a1, a2, a3, bl[sb][i][0], bl[sb][i][1]);
          }
        }
      }
    }
    if (r.flags & kSpanLast) {
      // join of the key warps' states through this stage, 8 rows of each row group
      // at a time
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[i][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
          if (gq == 0) mls[kw * ROWS + rows0 + 8 * i + 2 * tg + e] = make_float2(m[i][e], x);
        }
      named_bar_sync(1, 128);  // states published; every warp is done with the stage
      if (lane == 0) mbar_arrive(&q_empty[r.qbuf]);
      float* jb = reinterpret_cast<float*>(sk(st));  // [KW][8 RW][JP]
      constexpr int TPR = 16 / C::RW;                // threads per joined row
      const int jr = tid / TPR, part = tid % TPR;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (r.row0 + 8 * i >= r.rows) break;  // CTA-uniform
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = rows0 + 8 * i + 2 * tg + e;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < KW; ++w) top = fmaxf(top, mls[w * ROWS + row].x);
          // m = -inf: this warp saw no key of the row, and acc is 0
          const float a = m[i][e] == -INFINITY ? 0.f : ex2(m[i][e] - top);
          float* dst = jb + ((kw * C::RW + rw) * 8 + 2 * tg + e) * C::JP + gq;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            dst[16 * k] = acc[k][i][e] * a;
            dst[16 * k + 8] = acc[k][i][e + 2] * a;
          }
        }
        named_bar_sync(1, 128);
        const int lrow = (jr >> 3) * 8 * NT + 8 * i + (jr & 7);  // row of the segment
        if (r.row0 + lrow < r.rows) {
          const int64_t at = (int64_t)r.piece * ROWS + lrow;
          float* og = ss.part.o + at * D;
#pragma unroll
          for (int q4 = 0; q4 < D / 4 / TPR; ++q4) {
            const int d = (q4 * TPR + part) * 4;
            float4 sum = *reinterpret_cast<const float4*>(jb + jr * C::JP + d);
#pragma unroll
            for (int w = 1; w < KW; ++w) {
              const float4 x =
                  *reinterpret_cast<const float4*>(jb + (w * 8 * C::RW + jr) * C::JP + d);
              sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
            }
            *reinterpret_cast<float4*>(og + d) = sum;
          }
          if (part == 0) {
            float top = -INFINITY, ls = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w) top = fmaxf(top, mls[w * ROWS + lrow].x);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
              const float2 x = mls[w * ROWS + lrow];
              ls += x.y * (x.x == -INFINITY ? 0.f : ex2(x.x - top));  // a NaN sum stays NaN
            }
            ss.part.ml[at] = make_float2(top, ls);
          }
        }
        named_bar_sync(1, 128);  // the buffer (and, last, the states) may be rewritten
      }
      fence_proxy_async_smem();
    }
    __syncwarp();
    if (lane == 0 && g >= 0) mbar_arrive(&empty[st]);
  }
  if (ss.beside) grid_dependency_wait();
}

}  // namespace pdb
