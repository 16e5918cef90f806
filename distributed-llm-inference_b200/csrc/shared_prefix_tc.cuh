// The prefix's spans on the 5th-generation tensor cores (tcgen05 + TMEM + TMA,
// sm_100a, FP16, head_dim 64 / 128, block_size % 16 == 0).
//
// All B T G rows of a kv head see the whole prefix, so this is a dense product
// pair per kv head: S = Q K^T, O = P V with M = B T G. An item is (kv head,
// pair of 128-row query tiles); all items have the same number of 128-key
// tiles. With few items each is cut into `splits` ranges, one per CTA; else the
// (item, key tile) units are cut into one contiguous range per CTA of equal
// length, and a CTA works on the end of one item and the start of the next (a
// second piece costs it a second set of queries and a second epilogue, 5 us). CTA
// c's piece of item i is piece i + c of the partials.
//
// One CTA per SM, eleven warps:
//   * warps 0-3 and 4-7: softmax of query tile 0 and 1, one row per thread: read
//     the S row from TMEM, base-2 softmax against a running maximum that is
//     raised only when a logit passes it by 2^8 (O in TMEM is rescaled then;
//     exact after the final division), write P in two FP16 terms over S in TMEM.
//   * warps 9 and 10: TMA, for K and for V (one warp issues a 16-row box every
//     ~100 cycles, the TMA unit takes one every 61). K and V tiles (128 keys) go
//     through one ring of buffers in the order K0 V0 K1 V1 ..
//   * warp 8: MMA issuer (warp-uniform, one elected lane). Per key tile j:
//     O0 += P0 V_j, S0 = Q0 K_{j+1}, O1 += P1 V_j, S1 = Q1 K_{j+1}: while one
//     tile's rows are exponentiated the tensor cores work for the other.
//     The MMAs of a CTA run in issue order, so S_{j+1} may overwrite P_j
//     without a barrier, and the commit that publishes S_{j+1} also says that
//     O holds P_j V_j (what a rescale needs).
// Measured on 4096 rows x 8192 keys x 8 heads, 128 dims: 178 us with the join, 0.77 PFLOP/s
// of the formula's operations and half as many again for the second term of P (147 us without
// it); tensor pipe 65% busy. Handing P over in halves (the product of one while the other is exponentiated) or
// reading the logits a quarter ahead were slower (190 to 200), as was rounding the first term
// and converting it back (190).
// TMEM: S0 S1 O0 O1, 128 columns each = all 512.
// Query rows: a tile holds floor(128 / G) tokens with all G heads of the kv
// head, one TMA box {64 columns, G heads, floor(128 / G) tokens}, so any group
// size fills the tile up to its remainder.
// Bound: a row tile's chain of softmax (128 exponentials and their two terms per thread),
// P V and the next Q K^T, two of which overlap. The tensor cores alone take 6 x 512 cycles
// per two row tiles and key tile, the exponentials 2 x 128 x 128 at 16 a cycle = 2048.
#pragma once

#include "shared_prefix_mma.cuh"

namespace pdb {

struct PrefixTcParams {
  const int32_t* table;
  int2* dir;                  // [items] first, last CTA
  float2* ml;                 // [pieces][256]
  float* o;                   // [pieces][256][D]
  int64_t num_blocks;
  int tokens;                 // B T
  int H, KVH, G;
  int per_tile;               // tokens per 128-row tile
  int pairs;                  // pairs of query tiles per kv head
  int key_tiles;              // 128-key tiles of the prefix
  int splits;                 // ranges per item, or 0: equal ranges over all units
  int prefix_length, block_size, bs_shift;
  float scale_log2;
};

template <int D>
struct PrefixTc {
  static constexpr int BM = 128, BN = 128;
  static constexpr int HALVES = D / 64, UNITS = BN / 16;
  static constexpr int Q_BYTES = BM * D * 2, KV_BYTES = BN * D * 2;
  static constexpr int BUFS = D == 128 ? 5 : 8;  // ring of K and V tiles
  static constexpr int THREADS = 352;
  static constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = 256;
  static constexpr int NBARS = 2 * BUFS + 1 + 2 + 2 + 2 + 1;
  static constexpr size_t SMEM = 1024 + 2 * (size_t)Q_BYTES + (size_t)BUFS * KV_BYTES + NBARS * 8 + 16;
};

// Logits of keys at or past `valid` (of 64): -inf.
__device__ __forceinline__ void mask64(uint32_t* s, int valid) {
  if (valid < 64) {
#pragma unroll
    for (int x = 0; x < 64; ++x)
      if (x >= valid) s[x] = __float_as_uint(-INFINITY);
  }
}
__device__ __forceinline__ float max64(const uint32_t* s) {
  float mx[8];
#pragma unroll
  for (int y = 0; y < 8; ++y) mx[y] = __uint_as_float(s[y]);
#pragma unroll
  for (int x = 8; x < 56; x += 16)
#pragma unroll
    for (int y = 0; y < 8; ++y)
      mx[y] = fmax3(mx[y], __uint_as_float(s[x + y]), __uint_as_float(s[x + 8 + y]));
#pragma unroll
  for (int y = 0; y < 8; ++y) mx[y] = fmaxf(mx[y], __uint_as_float(s[56 + y]));
  return fmax3(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
}
// The weights 2^(c s - ref) of 64 keys in two FP16 terms, as pairs: of each 32 keys
// pk[0 .. 15] the first 11 bits (cut off, so that the rest is exact), pk[16 .. 31] the rest,
// rounded to 11 bits. Together 2^-21 of a weight is lost at most (2^-25 in all below
// 2^-14, where FP16 thins out; a row's largest weight is 1 at least). One rounded FP16 number
// is off by 2^-11 of a weight, as much as rounding the output adds. Returns the weights' sum in FP32.
__device__ __forceinline__ float weights64(const uint32_t* s, uint32_t* pk, float c, float ref) {
  const uint64_t c2 = f2(c, c), nm2 = f2(-ref, -ref), minus = f2(-1.f, -1.f);
  uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int x = 0; x < 32; ++x) {
    float y0, y1;
    f2_split(ffma2(f2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1])), c2, nm2), y0, y1);
    const float a = ex2(y0), b = ex2(y1);
    const uint64_t w = f2(a, b);
    sum[x & 3] = fadd2(sum[x & 3], w);
    const float ah = __uint_as_float(__float_as_uint(a) & 0xffffe000u);
    const float bh = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
    pk[(x & 16) + x] = pack_half2(ah, bh);
    f2_split(ffma2(f2(ah, bh), minus, w), y0, y1);
    pk[(x & 16) + 16 + x] = pack_half2(y0, y1);
  }
  float r[8];
#pragma unroll
  for (int x = 0; x < 4; ++x) f2_split(sum[x], r[2 * x], r[2 * x + 1]);
  return ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
}

template <int D>
__global__ void __launch_bounds__(PrefixTc<D>::THREADS, 1)
prefix_tc_kernel(const PrefixTcParams p, const __grid_constant__ CUtensorMap qmap,
                 const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = PrefixTc<D>;
  constexpr int BM = C::BM, BN = C::BN, HALVES = C::HALVES, UNITS = C::UNITS, BUFS = C::BUFS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto sq = [&](int i) { return base + (size_t)i * C::Q_BYTES; };
  auto buf = [&](int i) { return base + 2 * C::Q_BYTES + (size_t)i * C::KV_BYTES; };
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + 2 * C::Q_BYTES + (size_t)BUFS * C::KV_BYTES);
  uint64_t* full = bars;           // [BUFS] tile landed
  uint64_t* empty = bars + BUFS;   // [BUFS] both products that read it are done (commit)
  uint64_t* q_full = empty + BUFS;     // the piece's query tiles landed
  uint64_t* s_full = q_full + 1;       // [2] S of tile i in TMEM (commit)
  uint64_t* p_full = s_full + 2;       // [2] P of tile i in TMEM (4 arrivals)
  uint64_t* o_full = p_full + 2;       // [2] the piece's last product of tile i is done (commit)
  uint64_t* piece_done = o_full + 2;   // both softmax groups have read O (8 arrivals)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBARS);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(piece_done, 8);
    fence_barrier_init();
  }
  grid_dependency_wait();
  launch_dependents();
  if (warp == 0) {
    tc_alloc(tmem_slot, C::TMEM_COLS);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool live = true;  // after one expired wait a thread stops waiting
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (live) live = mbar_wait(bar, parity);
  };

  // this CTA's units [u0, u1) of (item, key tile)
  const int units = p.KVH * p.pairs * p.key_tiles;
  const int ctas = unit_ctas(units, (int)gridDim.x), me = (int)blockIdx.x;
  int u0, u1;
  if (p.splits) {
    const int it = me / p.splits, part = me - it * p.splits;
    u0 = it * p.key_tiles + unit_begin(part, p.key_tiles, p.splits);
    u1 = it * p.key_tiles + unit_begin(part + 1, p.key_tiles, p.splits);
  } else {
    u0 = unit_begin(me, units, ctas);
    u1 = unit_begin(me + 1, units, ctas);
  }
  // Piece that starts at unit u: item, first key tile, number of key tiles.
  auto piece = [&](int u, int& item, int& j0, int& nj) {
    item = u / p.key_tiles;
    j0 = u - item * p.key_tiles;
    const int end = (item + 1) * p.key_tiles;
    nj = (end < u1 ? end : u1) - u;
  };
  // Tiles that hold rows: a kv head's last pair may lack its second.
  auto tiles_of = [&](int pair) { return (2 * pair + 1) * p.per_tile < p.tokens ? 2 : 1; };

  if (warp >= 9) {
    // ---- TMA: warp 9 the queries and K tiles, warp 10 the V tiles -------------------
    const int kv = warp - 9;
    const CUtensorMap* map = kv ? &vmap : &kmap;
    int g = kv, n = 0;  // ring position (K and V alternate), pieces so far
    int item, j0, nj;
    // Pool row of this lane's unit of key tile j: -1 past the end or without a page.
    auto look_up = [&](int j) -> int {
      const int t = j * BN + lane * 16;
      if (lane >= UNITS || t >= p.prefix_length) return -1;
      const int pi = p.bs_shift >= 0 ? t >> p.bs_shift : t / p.block_size;
      const int page = __ldg(p.table + pi);
      if (page < 0 || (int64_t)page >= p.num_blocks) {
        raise_error(0x1u);
        return -1;
      }
      return page * p.block_size + (t - pi * p.block_size);
    };
    for (int u = u0; u < u1; u += nj, ++n) {
      piece(u, item, j0, nj);
      const int h = item / p.pairs, pair = item % p.pairs, nt = tiles_of(pair);
      int next = look_up(j0);
      if (kv == 0) {
        // the query buffers double as the epilogue's staging: free once it is done
        if (n > 0) wait(piece_done, (uint32_t)(n - 1) & 1u);
        if (lane == 0) {
          if (j0 == 0) p.dir[item].x = me;
          if (j0 + nj == p.key_tiles) p.dir[item].y = me;
          mbar_arrive_expect_tx(q_full, (uint32_t)(nt * HALVES * p.per_tile * p.G * 128));
          for (int i = 0; i < nt; ++i)
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_3d(sq(i) + hf * (BM * 128), &qmap, hf * 64, h * p.G,
                          (2 * pair + i) * p.per_tile, q_full);
        }
        __syncwarp();
      }
      for (int j = j0; j < j0 + nj; ++j, g += 2) {
        const int cell = next;
        if (j + 1 < j0 + nj) next = look_up(j + 1);  // in flight while this tile is issued
        const unsigned ok = __ballot_sync(0xffffffffu, cell >= 0);
        const int b = g % BUFS;
        if (g >= BUFS) wait(&empty[b], (uint32_t)(g / BUFS - 1) & 1u);
        if (ok != (1u << UNITS) - 1) {  // units without a page (past the end, or bad): zeros
          for (int i = lane; i < UNITS * 16 * (D / 8); i += 32) {
            const int row = i / (D / 8), c = i % (D / 8);
            if (!(ok >> (row >> 4) & 1))
              *reinterpret_cast<uint4*>(buf(b) + (c >> 3) * (BN * 128) + row * 128 +
                                        ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        int from[UNITS];
#pragma unroll
        for (int i = 0; i < UNITS; ++i) from[i] = __shfl_sync(0xffffffffu, cell, i);
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[b], (uint32_t)__popc(ok) * HALVES * 2048u);
#pragma unroll
          for (int i = 0; i < UNITS; ++i) {
            if (from[i] < 0) continue;
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
              tma_load_3d(buf(b) + hf * (BN * 128) + i * 2048, map, hf * 64, h, from[i], &full[b]);
          }
        }
        __syncwarp();
      }
    }
    // every commit to an `empty` barrier has arrived before the CTA ends
    const int used = g - kv;  // tiles of both kinds
    for (int gg = used > BUFS ? used - BUFS : 0; gg < used; ++gg)
      wait(&empty[gg % BUFS], (uint32_t)(gg / BUFS) & 1u);
  } else if (warp == 8) {
    // ---- MMA issuer -------------------------------------------------------------
    constexpr uint32_t IDESC_S = f16_idesc(BM, BN, 0, 0);
    constexpr uint32_t IDESC_O = f16_idesc(BM, D, 0, 1);
    const uint64_t q_desc = sw128_desc(smem_u32(sq(0)), 16, 1024);
    const uint64_t k_desc = sw128_desc(smem_u32(buf(0)), 16, 1024);
    const uint64_t v_desc = sw128_desc(smem_u32(buf(0)), BN * 128, 1024);
    constexpr uint64_t STEP = C::KV_BYTES >> 4, Q_STEP = C::Q_BYTES >> 4;
    auto qk = [&](int i, int b) {  // S_i = Q_i K
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t qo = (uint64_t)((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4;
        const uint64_t ko = (uint64_t)((kk >> 2) * (BN * 128) + (kk & 3) * 32) >> 4;
        tc_mma_elect(tmem + C::S_COL + i * 128, q_desc + i * Q_STEP + qo, k_desc + b * STEP + ko,
                     IDESC_S, kk > 0 ? 1u : 0u);
      }
      tc_commit_elect(&s_full[i]);
    };
    int g = 0, n = 0, tile[2] = {0, 0};  // ring position, pieces, P tiles so far
    int item, j0, nj;
    for (int u = u0; u < u1; u += nj, ++n) {
      piece(u, item, j0, nj);
      const int nt = tiles_of(item % p.pairs);
      wait(q_full, (uint32_t)n & 1u);
      // O of the previous piece has been read (the TMA warp waited for it
      // before it loaded these queries)
      wait(&full[g % BUFS], (uint32_t)(g / BUFS) & 1u);
      __syncwarp();
      tc_fence_after();
      for (int i = 0; i < nt; ++i) qk(i, g % BUFS);
      tc_commit_elect(&empty[g % BUFS]);
      ++g;  // now at V of the first key tile
      for (int j = 0; j < nj; ++j) {
        const int vb = g % BUFS, kb = (g + 1) % BUFS;
        wait(&full[vb], (uint32_t)(g / BUFS) & 1u);
        const bool more = j + 1 < nj;
        for (int i = 0; i < nt; ++i) {
          wait(&p_full[i], (uint32_t)tile[i]++ & 1u);
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)  // 16 keys: both terms of P
#pragma unroll
            for (int term = 0; term < 2; ++term)
              tc_mma_ts_elect(tmem + C::O_COL + i * 128,
                              tmem + C::S_COL + i * 128 + (kk >> 1) * 32 + term * 16 + (kk & 1) * 8,
                              v_desc + vb * STEP + kk * (16 * 128 >> 4), IDESC_O,
                              (j > 0 || kk + term > 0) ? 1u : 0u);
          if (!more) tc_commit_elect(&o_full[i]);
          if (i == nt - 1) tc_commit_elect(&empty[vb]);
          if (more) {
            if (i == 0) {
              wait(&full[kb], (uint32_t)((g + 1) / BUFS) & 1u);
              __syncwarp();
              tc_fence_after();
            }
            qk(i, kb);
          }
        }
        if (more) tc_commit_elect(&empty[kb]);
        g += more ? 2 : 1;
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread owns row `lane_row` of query tile `i` ---------------------
    const int i = warp >> 2, wq = warp & 3, lane_row = wq * 32 + lane;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const uint32_t s_col = tmem + lane_base + C::S_COL + i * 128;
    const uint32_t o_col = tmem + lane_base + C::O_COL + i * 128;
    const float c = p.scale_log2;
    int n = 0, tile = 0, done = 0;  // pieces; this tile's S phases; its pieces
    int item, j0, nj;
    for (int u = u0; u < u1; u += nj, ++n) {
      piece(u, item, j0, nj);
      const int pair = item % p.pairs;
      if (i < tiles_of(pair)) {
        float m_used = -INFINITY, l = 0.f;
        // Round -1 of the first piece runs this code on what TMEM holds, while the
        // first tiles are on their way, and throws the result away: it brings the
        // code, whose first execution otherwise waits on instruction fetches.
        for (int j = n == 0 ? -1 : 0; j < nj; ++j) {
          const bool real = j >= 0;
          if (real) wait(&s_full[i], (uint32_t)tile & 1u);
          tc_fence_after();
          // Pass 1: the row's maximum. The second half of the logits stays in
          // registers, the first is read again: 128 at once would not fit.
          const int valid = real ? p.prefix_length - (j0 + j) * BN : BN;
          uint32_t s[64];
          float top = -INFINITY;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            tc_ld32(s_col + hf * 64, s);
            tc_ld32(s_col + hf * 64 + 32, s + 32);
            tc_wait_ld();
            tc_reg_fence32(s);
            tc_reg_fence32(s + 32);
            mask64(s, valid - hf * 64);
            top = fmaxf(top, max64(s));
          }
          top *= c;
          float alpha = 1.f;
          if (top > m_used + 8.f) {
            alpha = ex2(m_used - top);
            m_used = top;
          }
          // all logits -inf so far: any finite reference gives weights 0
          const float ref = m_used == -INFINITY ? 0.f : m_used;
          // Pass 2: weights, second half first, the two terms of 32 keys over their own
          // logits (which are in registers by then).
          uint32_t pk[64];
          float sum = weights64(s, pk, c, ref);
          if (real) {
            tc_st32(s_col + 64, pk);
            tc_st32(s_col + 96, pk + 32);
          }
          tc_ld32(s_col, s);
          tc_ld32(s_col + 32, s + 32);
          tc_wait_ld();
          tc_reg_fence32(s);
          tc_reg_fence32(s + 32);
          mask64(s, valid);
          sum += weights64(s, pk, c, ref);
          l = l * alpha + sum;
          if (!real) {
            m_used = -INFINITY;
            l = 0.f;
            continue;
          }
          tc_st32(s_col, pk);
          tc_st32(s_col + 32, pk + 32);
          if (valid < BN && i == 0) {
            // V rows past the prefix (stale cells of its last unit): zeros. K and V
            // alternate in the ring: this tile's V is buffer 2 * tile + 1.
            // Tile 0 always runs, and its product is issued first.
            const int g = 2 * tile + 1, b = g % BUFS;
            wait(&full[b], (uint32_t)(g / BUFS) & 1u);
            for (int x = lane_row; x < (BN - valid) * (D / 8); x += 128) {
              const int row = valid + x / (D / 8), cc = x % (D / 8);
              *reinterpret_cast<uint4*>(buf(b) + (cc >> 3) * (BN * 128) + row * 128 +
                                        (((cc & 7) ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            uint32_t ov[32];
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              tc_ld32(o_col + q * 32, ov);
              tc_wait_ld();
              tc_reg_fence32(ov);
#pragma unroll
              for (int x = 0; x < 32; ++x)
                ov[x] = __float_as_uint(__uint_as_float(ov[x]) * alpha);
              tc_st32(o_col + q * 32, ov);
            }
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[i]);
          ++tile;
        }
        // the piece's partial: O rows through this warp's quarter of the query
        // buffer, 64 columns at a time, so that stores cover whole row segments
        wait(&o_full[i], (uint32_t)done & 1u);
        ++done;
        tc_fence_after();
        const int64_t at0 = (int64_t)(item + me) * (2 * BM) + i * BM + wq * 32;
        const int token0 = (2 * pair + i) * p.per_tile;
        const int used_rows =
            (p.tokens - token0 < p.per_tile ? p.tokens - token0 : p.per_tile) * p.G;
        unsigned char* stage = sq(i) + wq * 32 * 256 * (D == 128 ? 1 : 0) + (D == 64 ? wq * 32 * 128 : 0);
        constexpr int COLS = D == 128 ? 64 : 32;  // fp32 columns per round: 8 / 4 KB per warp
        constexpr int CH = COLS / 4;              // 16-byte chunks of a staged row
#pragma unroll
        for (int q = 0; q < D / COLS; ++q) {
#pragma unroll
          for (int q2 = 0; q2 < COLS / 32; ++q2) {
            uint32_t ov[32];
            tc_ld32(o_col + q * COLS + q2 * 32, ov);
            tc_wait_ld();
            tc_reg_fence32(ov);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const int ch = q2 * 8 + x;
              *reinterpret_cast<uint4*>(stage + lane * (COLS * 4) + ((ch ^ (lane & 7)) << 4)) =
                  make_uint4(ov[4 * x], ov[4 * x + 1], ov[4 * x + 2], ov[4 * x + 3]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int x = 0; x < CH; ++x) {  // 32 rows x CH chunks
            const int e = x * 32 + lane, rr = e / CH, ch = e % CH;
            if (wq * 32 + rr < used_rows)
              *reinterpret_cast<uint4*>(p.o + (at0 + rr) * D + q * COLS + ch * 4) =
                  *reinterpret_cast<const uint4*>(stage + rr * (COLS * 4) + ((ch ^ (rr & 7)) << 4));
          }
          __syncwarp();
        }
        if (lane_row < used_rows) p.ml[at0 + lane] = make_float2(m_used, l);
        tc_fence_before();
        fence_proxy_async_smem();  // the staging writes, before the next query load
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(piece_done);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tc_dealloc(tmem, C::TMEM_COLS);
  }
}

}  // namespace pdb
