// Spans over FP32 pools on the warp-level tensor cores
// (sm_100a, head_dim 64 / 128, 16-byte rows), with FP32 accuracy.
//
// An FP32 number x is the sum of x1 = x rounded to the 11 bits of TF32 and of a rest
// x2 = x - x1 (exact), of which 11 bits are kept: 2^-21 |x| is lost at most. A product is
// then x1 y1 + x1 y2 + x2 y1, three TF32 products with sums in FP32; x2 y2, below
// 2^-22 |x y|, is left out. The tensor cores may cut sums off instead of rounding them, so
// no chain of theirs is long: the logits take two chains of D / 16 for x1 y1 and one
// for the small terms, the values one of each per tile of 32 keys, and tiles are added in
// FP32 by the multiply-add that also rescales the running O.
//
// One CTA per (row tile of RT, kv head, key range), as the FP32-pipe kernel, four
// warps: 16 rows and all keys of a tile each (KW = 1, RT = 64), or RT = 32 and 16 rows with
// the keys split over KW = 2 and 4 warps, joined at the end. A product
// m16n8k8 takes an SM's quarter 8.1 cycles (measured, as for FP16 with k = 16), so the
// three of them give 166 multiply-adds a cycle and SM at most. Measured: 512 rows of 8 kv heads
// over 4096 keys of 128 dims 204 us with the join, 331 on the FP32 pipes, whose reads of
// shared memory bound them; 64 x 8 spans of 16 rows and 512 keys 113 (259), of 32 rows 153 (303).
// It is bound by the issue of eight warps an SM: splitting an operand costs four instructions
// an element, a third of all, and the products wait for it.
//
// An infinity or NaN among K or V makes NaN of sums that FP32 arithmetic would keep
// (its rest is NaN, and 0 inf is NaN). Rows that come out with a NaN are computed a
// second time in plain FP32. A drafted token's V is also met by rows that must not see
// it: what is not finite in it is staged as 0, which leaves those rows as they are, and
// the rows that do see it are computed a second time.
#pragma once

#include "shared_prefix.cuh"

namespace pdb {

template <int D_, int KW_>
struct SpanTf32 {
  static constexpr int D = D_, KW = KW_, NT = 128, KT = 32;
  static constexpr int RT = 64 / KW;
  static constexpr int NB = KT / 8 / KW;  // 8-key blocks per warp and tile
  // Row pitches without bank conflicts: Q and K are read as 16 bytes of rows gq (two
  // per phase, 16 banks apart), V as 16 bytes of rows 2 tg (four per phase, 8 apart).
  static constexpr int LK = D + 16, LV = D + 4;
  static constexpr int JP = D + 4;  // row pitch of the join buffer
  static constexpr size_t SMEM = (size_t)(RT * LK + 2 * KT * (LK + LV) + 4 * 16 * 2 + RT + 1) * sizeof(float);
  static_assert(4 * 16 * JP <= 2 * KT * (LK + LV), "join buffer fits the key buffers");
};

// x = hi + lo, both TF32 (their low 13 bits are 0), up to 2^-21 |x|.
__device__ __forceinline__ void tf32_split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

__device__ __forceinline__ void mma_1688_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7},"
      " {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class C>
__global__ void __launch_bounds__(C::NT, 2)
prefix_tf32_kernel(const PrefixParams p, int prefix_tiles, int own_tiles) {
  constexpr int D = C::D, KW = C::KW, KT = C::KT, RT = C::RT, NB = C::NB, LK = C::LK, LV = C::LV,
                JP = C::JP, TPK = C::NT / KT;
  extern __shared__ __align__(16) float smem_f[];
  float* sq = smem_f;                                            // [RT][LK]
  float* sk = sq + RT * LK;                                      // [2][KT][LK]
  float* sv = sk + 2 * KT * LK;                                  // [2][KT][LV]
  float2* mls = reinterpret_cast<float2*>(sv + 2 * KT * LV);     // [4 warps][16 rows]
  int* redo = reinterpret_cast<int*>(mls + 4 * 16);              // [RT] rows of the second pass
  int* odd_key = redo + RT;                                      // first key staged as 0
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y, G = p.G;
  const int gq = lane >> 2, tg = lane & 3;
  const int kw = warp % KW, rows0 = warp / KW * 16;  // this warp's keys and rows
  const bool prefix = prefix_tiles > 0, beside = !prefix && p.beside;
  if (!beside) grid_dependency_wait();
  launch_dependents();
  const PartSet& set = prefix ? p.prefix : p.own;
  const SpanTile t = span_tile(p, set, prefix, own_tiles, RT);
  if (t.k0 >= t.k1) {
    if (beside) grid_dependency_wait();
    return;
  }
  const int k0 = t.k0, k1 = t.k1;
  auto global_row = [&](int row) {  // of q and out
    return (int64_t)(t.token0 + row / G) * p.H + (int64_t)h * G + row % G;
  };
  const float* kp = static_cast<const float*>(p.k_pool) + (int64_t)h * D;
  const float* vp = static_cast<const float*>(p.v_pool) + (int64_t)h * D;
  // Four threads stage a key. Its page is read one tile ahead and looked at only when
  // the key is staged, so that no thread waits for the read.
  const int sj = tid / TPK, sc = tid % TPK * 4;
  auto page_of = [&](int t0) {
    const int pi = p.bs_shift >= 0 ? (t0 + sj) >> p.bs_shift : (t0 + sj) / p.block_size;
    return t0 + sj < k1 && pi < t.width ? __ldg(t.table + pi) : -1;
  };
  auto cell_of = [&](int t0, int page) -> int64_t {
    if (t0 + sj >= k1) return -1;
    if (page < 0 || (int64_t)page >= p.num_blocks) {
      raise_error(0x1u);
      return -1;
    }
    return (int64_t)page * p.block_size +
           (p.bs_shift >= 0 ? (t0 + sj) & (p.block_size - 1) : (t0 + sj) % p.block_size);
  };
  auto stage = [&](int64_t cell, int buf) {  // no page, past the end: zeros
    float* dk = sk + (buf * KT + sj) * LK + sc;
    float* dv = sv + (buf * KT + sj) * LV + sc;
    const int64_t at = cell < 0 ? 0 : cell * p.KVH * D + sc;
#pragma unroll
    for (int c = 0; c < D; c += TPK * 4) {
      cp_async16(dk + c, kp + at + c, cell >= 0);
      cp_async16(dv + c, vp + at + c, cell >= 0);
    }
    cp_async_commit();
  };
  // the queries ride on the first tile's group; rows past the item's: zeros
  const float* q = static_cast<const float*>(p.q);
#pragma unroll 4
  for (int i = tid; i < RT * (D / 4); i += C::NT) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const bool in = t.r0 + r < t.rend;
    cp_async16(sq + r * LK + d, q + (in ? global_row(t.r0 + r) * D + d : 0), in);
  }
  stage(cell_of(k0, page_of(k0)), 0);
  int page = page_of(k0 + KT);
  for (int i = tid; i < RT; i += C::NT) redo[i] = 0;
  if (tid == 0) *odd_key = INT_MAX;
  __syncthreads();  // before any thread marks a key
  int row[2], limit[2];  // rows of the item; keys [0, limit) are seen
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    row[e] = t.r0 + rows0 + gq + 8 * e;
    limit[e] = row[e] >= t.rend ? -1 : prefix ? k1 : min(prefix_limit(t.n, t.count, row[e] / G), k1);
  }
  float* logits = p.logits && t.b >= 0
                      ? p.logits + ((int64_t)t.b * p.KVH + h) * p.logits_width * p.T * G
                      : nullptr;
  const float* q_l = sq + (rows0 + gq) * LK + 4 * tg;
  float m[2], l[2], acc[D / 32][4][4];  // dims 32 j + 4 column + i of rows gq, gq + 8

  for (bool plain = false;; plain = true) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m[e] = -INFINITY, l[e] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = 0.f;
    int buf = 0;
    for (int t0 = k0; t0 < k1; t0 += KT, buf ^= 1) {
      if (t0 + KT < k1) {
        stage(cell_of(t0 + KT, page), buf ^ 1);
        page = page_of(t0 + 2 * KT);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      if (!plain && !prefix && t0 + sj > t.n - t.count && t0 + sj < k1) {  // this thread's pieces
        float* v = sv + (buf * KT + sj) * LV + sc;
        for (int c = 0; c < D; c += TPK * 4)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((__float_as_uint(v[c + e]) & 0x7f800000u) == 0x7f800000u) {
              v[c + e] = 0.f;
              atomicMin(odd_key, t0 + sj);
            }
      }
      __syncthreads();
      const float* ck = sk + (buf * KT + kw * NB * 8) * LK;
      const float* cv = sv + (buf * KT + kw * NB * 8) * LV;
      const int key0 = t0 + kw * NB * 8;
      // S: keys key0 + 8 i + 2 tg + (e & 1) of rows gq + 8 (e >> 1)
      float s[NB][4];
      if (!plain) {
        float big[2][NB][4], small[NB][4];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) big[0][i][e] = big[1][i][e] = small[i][e] = 0.f;
        // a 16-byte piece of a row is dims 4 tg .. of two products: which dim is which
        // k of a product does not matter as long as both operands agree
#pragma unroll 2
        for (int d = 0; d < D; d += 16) {
          const float4 x = *reinterpret_cast<const float4*>(q_l + d);
          const float4 y = *reinterpret_cast<const float4*>(q_l + 8 * LK + d);
          uint32_t ah[2][4], al[2][4];
          tf32_split(x.x, ah[0][0], al[0][0]);
          tf32_split(y.x, ah[0][1], al[0][1]);
          tf32_split(x.y, ah[0][2], al[0][2]);
          tf32_split(y.y, ah[0][3], al[0][3]);
          tf32_split(x.z, ah[1][0], al[1][0]);
          tf32_split(y.z, ah[1][1], al[1][1]);
          tf32_split(x.w, ah[1][2], al[1][2]);
          tf32_split(y.w, ah[1][3], al[1][3]);
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const float4 k4 = *reinterpret_cast<const float4*>(ck + (8 * i + gq) * LK + d + 4 * tg);
            uint32_t bh[4], bl[4];
            tf32_split(k4.x, bh[0], bl[0]);
            tf32_split(k4.y, bh[1], bl[1]);
            tf32_split(k4.z, bh[2], bl[2]);
            tf32_split(k4.w, bh[3], bl[3]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              mma_1688_tf32(big[u][i], ah[u], bh[2 * u], bh[2 * u + 1]);
              mma_1688_tf32(small[i], ah[u], bl[2 * u], bl[2 * u + 1]);
              mma_1688_tf32(small[i], al[u], bh[2 * u], bh[2 * u + 1]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = big[0][i][e] + big[1][i][e] + small[i][e];
      } else {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float* x = sq + (rows0 + gq + 8 * (e >> 1)) * LK;
            const float* y = ck + (8 * i + 2 * tg + (e & 1)) * LK;
            float sum = 0.f;
#pragma unroll 1
            for (int d = 0; d < D; ++d) sum = fmaf(x[d], y[d], sum);
            s[i][e] = sum;
          }
      }
      float mx[2] = {-INFINITY, -INFINITY}, alpha[2], ref[2];
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * i + 2 * tg + (e & 1);
          const bool seen = key < limit[e >> 1];
          s[i][e] = seen ? s[i][e] * p.scale_log2 : -INFINITY;
          if (logits && seen && (!plain || redo[rows0 + gq + 8 * (e >> 1)])) logits[(int64_t)key * p.T * G + row[e >> 1]] = s[i][e];
          mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        const float mn = fmaxf(m[e], mx[e]);
        alpha[e] = mn == -INFINITY ? 1.f : exp2f(m[e] - mn);  // m = -inf: 0
        ref[e] = mn == -INFINITY ? 0.f : mn;
        m[e] = mn;
        l[e] *= alpha[e];
      }
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = exp2f(s[i][e] - ref[e >> 1]);
          l[e >> 1] += s[i][e];
        }
      if (!plain) {
        // P as the left operand: k of a product = keys 2 tg, 2 tg + 1, as S lies
        uint32_t ph[NB][4], pl[NB][4];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          tf32_split(s[i][0], ph[i][0], pl[i][0]);
          tf32_split(s[i][2], ph[i][1], pl[i][1]);
          tf32_split(s[i][1], ph[i][2], pl[i][2]);
          tf32_split(s[i][3], ph[i][3], pl[i][3]);
        }
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          float big[4][4], small[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) big[i][e] = small[i][e] = 0.f;
#pragma unroll
          for (int kb = 0; kb < NB; ++kb) {
            const float* v_l = cv + (8 * kb + 2 * tg) * LV + 32 * j + 4 * gq;
            const float4 x = *reinterpret_cast<const float4*>(v_l);
            const float4 y = *reinterpret_cast<const float4*>(v_l + LV);
            const float v0[4] = {x.x, x.y, x.z, x.w}, v1[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t h0, l0, h1, l1;
              tf32_split(v0[i], h0, l0);
              tf32_split(v1[i], h1, l1);
              mma_1688_tf32(big[i], ph[kb], h0, h1);
              mma_1688_tf32(small[i], ph[kb], l0, l1);
              mma_1688_tf32(small[i], pl[kb], h0, h1);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[j][i][e] = fmaf(acc[j][i][e], alpha[e >> 1], big[i][e] + small[i][e]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][i][e] *= alpha[e >> 1];
#pragma unroll 1
        for (int key = 0; key < 8 * NB; ++key) {
          float w0 = 0.f, w1 = 0.f;  // the key's weights in rows gq, gq + 8
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (key >> 3 == i && (key & 1) == e) w0 = s[i][e], w1 = s[i][e + 2];
          w0 = __shfl_sync(0xffffffffu, w0, (lane & ~3) | ((key & 7) >> 1));
          w1 = __shfl_sync(0xffffffffu, w1, (lane & ~3) | ((key & 7) >> 1));
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float x = cv[key * LV + 32 * j + 4 * (2 * tg + e) + i];
                if (w0 != 0.f) acc[j][i][e] = fmaf(w0, x, acc[j][i][e]);
                if (w1 != 0.f) acc[j][i][e + 2] = fmaf(w1, x, acc[j][i][e + 2]);
              }
        }
      }
      __syncthreads();  // the buffer may be staged again
    }
    if (!plain) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        bool odd = limit[e] > *odd_key;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            odd |= acc[j][i][2 * e] != acc[j][i][2 * e] || acc[j][i][2 * e + 1] != acc[j][i][2 * e + 1];
        if (odd && row[e] < t.rend) redo[rows0 + gq + 8 * e] = 1;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    if constexpr (KW == 1) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (row[e] >= t.rend || (plain && !redo[rows0 + gq + 8 * e])) continue;
        const int64_t at = (int64_t)t.slot * p.rows + global_row(row[e]);
        if (tg == 0) set.ml[at] = make_float2(m[e], l[e]);
        float* o = set.o + at * D + 8 * tg;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            *reinterpret_cast<float4*>(o + 32 * j + 4 * c) =
                make_float4(acc[j][0][c + 2 * e], acc[j][1][c + 2 * e], acc[j][2][c + 2 * e],
                            acc[j][3][c + 2 * e]);
      }
    } else {
      // join of the warps that share rows, through the key buffers
      float* jb = sk;  // [4 warps][16 rows][JP]
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (tg == 0) mls[warp * 16 + gq + 8 * e] = make_float2(m[e], l[e]);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < KW; ++w) top = fmaxf(top, mls[(warp / KW * KW + w) * 16 + gq + 8 * e].x);
        const float a = m[e] == -INFINITY ? 0.f : exp2f(m[e] - top);  // -inf: no key, acc is 0
        float* o = jb + (warp * 16 + gq + 8 * e) * JP + 8 * tg;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            *reinterpret_cast<float4*>(o + 32 * j + 4 * c) =
                make_float4(acc[j][0][c + 2 * e] * a, acc[j][1][c + 2 * e] * a,
                            acc[j][2][c + 2 * e] * a, acc[j][3][c + 2 * e] * a);
      }
      __syncthreads();
      for (int i = tid; i < RT * (D / 4); i += C::NT) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, w0 = r / 16 * KW;
        if (t.r0 + r >= t.rend) break;
        if (plain && !redo[r]) continue;
        const int64_t at = (int64_t)t.slot * p.rows + global_row(t.r0 + r);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(jb + ((w0 + w) * 16 + r % 16) * JP + d);
          sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
        }
        *reinterpret_cast<float4*>(set.o + at * D + d) = sum;
        if (d == 0) {
          float top = -INFINITY, ls = 0.f;
#pragma unroll
          for (int w = 0; w < KW; ++w) top = fmaxf(top, mls[(w0 + w) * 16 + r % 16].x);
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            const float2 x = mls[(w0 + w) * 16 + r % 16];
            ls += x.y * (x.x == -INFINITY ? 0.f : exp2f(x.x - top));
          }
          set.ml[at] = make_float2(top, ls);
        }
      }
    }
    if (plain) break;
    __syncthreads();  // flags written, join buffer read
    bool any = false;
    for (int i = tid; i < RT; i += C::NT) any |= redo[i] != 0;
    if (!__syncthreads_or(any)) break;
    stage(cell_of(k0, page_of(k0)), 0);
    page = page_of(k0 + KT);
  }
  if (beside) grid_dependency_wait();
}

}  // namespace pdb
