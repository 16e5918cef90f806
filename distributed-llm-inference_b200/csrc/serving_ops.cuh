// C entry points of the shared-prefix attention, the verification of drafted
// tokens and the cache eviction: argument checks, kernel selection, workspace
// layout and launches. Included by paged_decode.cu, whose helpers it uses.
#pragma once

#include <algorithm>

#include "shared_prefix.cuh"
#include "shared_prefix_mma.cuh"
#include "shared_prefix_tf32.cuh"
#include "shared_prefix_tc.cuh"
#include "verify.cuh"
#include "evict.cuh"

namespace {

int page_shift(int64_t bs) {
  return (bs & (bs - 1)) == 0 ? __builtin_ctzll((unsigned long long)bs) : -1;
}

// ---- shared-prefix attention -------------------------------------------------
// The kernel of one key set: those with key ranges as slots (FP32 pipes, TF32, few rows),
// mma.sync over FP16, tcgen05.
enum SpanKernel { kSpanNone = 0, kSpanSlots, kSpanMma, kSpanTc };

struct PrefixPlan {
  int prefix_kernel, own_kernel;
  int nt;      // kSpanMma: 8-row tiles per segment
  int splits;  // kSpanTc: ranges per item, or 0
  pdb::PartSet prefix, own;
  size_t prefix_ml, prefix_o, prefix_dir, own_ml, own_o, own_dir, lse_off, logits_off, total;
};

// Rows per CTA of the FP32-pipe kernel, and of the TF32 kernel. Key ranges are cut for
// the latter's.
int simt_rows(int64_t rows) { return rows <= 8 ? 8 : rows <= 128 ? 32 : 64; }
int slot_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

// Key ranges for the FP32 kernel: a multiple of 64 keys, no shorter than
// `least`, so that `tiles` CTAs per range reach `want` CTAs where the keys allow.
void split_keys(int64_t keys, int64_t tiles, int64_t want, int64_t least, pdb::PartSet* s) {
  int64_t n = (want + tiles - 1) / tiles;
  const int64_t most = (keys + least - 1) / least;
  if (n > most) n = most;
  if (n < 1) n = 1;
  int64_t c = (keys + n - 1) / n;
  c = (c + 63) / 64 * 64;
  s->kind = pdb::kPartSlots;
  s->chunk = (int)c;
  s->slots = (int)((keys + c - 1) / c);
}
// Ranges of a prefix of `keys` keys over FP32 pools: the number with the earliest end if
// two CTAs an SM work in waves and a CTA's start takes as long as 64 keys. (8 kv heads of
// 128 dims, 4096 keys, 32 rows: 28 us with the 32 ranges of this rule, 39 with the 64 that
// four CTAs an SM would be; 512 rows: 207 with 4 in one wave, 204 with 10 in three.)
int64_t prefix_slots(int sms, int64_t tiles, int64_t keys) {
  int64_t best = 1, cost = -1;
  for (int64_t n = 1; n <= (keys + 63) / 64 && (n == 1 || tiles * n <= 4 * (int64_t)sms); ++n) {
    const int64_t waves = (tiles * n + 2 * sms - 1) / (2 * sms);
    const int64_t c = waves * (((keys + n - 1) / n + 63) / 64 * 64 + 64);
    if (cost < 0 || c < cost) {
      best = n;
      cost = c;
    }
  }
  return best;
}
// Rows per segment of the mma.sync kernel, in tiles of 8: the K and V tiles are
// read once per segment, so as many rows as there are, up to 32 (registers).
int span_nt(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

constexpr int kSpanCtasPerSm = 2;
// From this many rows on, a prefix goes to the tcgen05 kernel (128-row tiles);
// below, it is one more key set of the mma.sync kernel's launch.
constexpr int64_t kTcRows = 33;

// Ranges per item of the tcgen05 kernel (items: query tile pairs of all kv heads, with
// `tiles` key tiles each) when the mma.sync kernel runs beside it on the SMs that
// are left: those with the earlier end by the measured rates, or 0 where one after
// the other on all SMs ends no later. A key tile takes 2.6 us (head_dim 64: 1.9) after
// 8 us of start and end; 64 keys of own contexts 0.74 us of an SM's time at 16 rows
// or less, 1.2 at 32 (head_dim 64: 0.62), after 9 us. Own lengths are on the device:
// half the bound is taken. (B200: one token for 64 sequences over a prefix of 4096,
// 8 items: 55 us in turn, 45, 39, 38 and 39 with 3, 4, 5 and 6 ranges; 24 sequences
// of 6 tokens over 2501, 24 items: 40 in turn, 47, 42, 45 with 2, 3, 4; 128 of 5 tokens and
// 9 heads of 64 dims over 1999: 38 in turn, 48, 35, 37 with 1, 2, 3. Over 14 shapes the
// rule's choice costs 2% more than the best on average, 8% at most.)
int tc_splits(int sms, int64_t items, int64_t tiles, double own_units, int64_t own_rows, int64_t D) {
  const double tile = D == 128 ? 2.6 : 1.9;
  const double own = own_units * (D == 64 ? 0.62 : own_rows <= 16 ? 0.74 : 1.2);
  const int64_t all = sms / items < 1 ? 1 : sms / items;
  const double tc_all = items * all <= sms ? (double)((tiles + all - 1) / all)
                                           : (double)(items * tiles) / sms;
  double best = 8 + tile * tc_all + 10 + own / sms;
  int splits = 0;
  for (int64_t k = 1; k <= tiles && items * k < sms; ++k) {
    const double a = 8 + tile * ((tiles + k - 1) / k), b = 9 + own / (sms - items * k);
    if ((a > b ? a : b) < best) {
      best = a > b ? a : b;
      splits = (int)k;
    }
  }
  return splits;
}

PrefixPlan prefix_plan(int sms, int64_t B, int64_t T, int64_t H, int64_t KVH, int64_t D, int64_t P,
                       int64_t max_length, bool scored, bool tensor_cores, int impl) {
  PrefixPlan pl{};
  const int64_t G = H / KVH, TG = T * G, rows = B * T * H, all = B * TG;
  pl.prefix_kernel = P <= 0 ? kSpanNone : kSpanSlots;
  pl.own_kernel = max_length <= 0 ? kSpanNone : kSpanSlots;
  // unit and segment counts are 32-bit in the tensor-core kernels
  if (B * KVH * T * G * ((P + 63) / 64 + (max_length + 63) / 64 + 2) >= (int64_t(1) << 31))
    tensor_cores = false;
  if (tensor_cores && impl != PDB_PREFIX_SIMT) {
    if (pl.own_kernel) pl.own_kernel = kSpanMma;
    if (pl.prefix_kernel) {
      const bool tc = G <= 128 && (impl == PDB_PREFIX_TCGEN05 ||
                                   (impl == PDB_PREFIX_AUTO && all >= kTcRows));
      pl.prefix_kernel = tc ? kSpanTc : kSpanMma;
    }
  }
  size_t prefix_parts = 0, own_parts = 0, span_segments = 0;  // own_parts: of the mma.sync launch
  int beside_sms = 0;
  if (pl.prefix_kernel == kSpanSlots) {
    const int64_t tiles = (all + slot_rows(all) - 1) / slot_rows(all) * KVH;
    split_keys(P, tiles, tiles * prefix_slots(sms, tiles, P), 64, &pl.prefix);
    prefix_parts = (size_t)pl.prefix.slots * rows;
  } else if (pl.prefix_kernel == kSpanTc) {
    pdb::PartSet& s = pl.prefix;
    s.kind = pdb::kPartUnits;
    s.R = 256;
    s.half = (int)(128 / G);
    s.segments = (int)((B * T + 2 * s.half - 1) / (2 * s.half));
    const int64_t items = KVH * s.segments, tiles = (P + 127) / 128;
    if (pl.own_kernel == kSpanMma) {
      const int64_t r = 8 * span_nt(TG);
      pl.splits = tc_splits(sms, items, tiles,
                            (double)(B * KVH * ((TG + r - 1) / r)) * (max_length / 128.0 + 0.3), r, D);
      beside_sms = (int)items * pl.splits;
    }
    if (!pl.splits && items <= sms / 2)  // on all SMs: whole ranges where items are few
      pl.splits = (int)std::min<int64_t>(sms / items, tiles);
    s.grid = (int)(pl.splits ? items * pl.splits : std::min<int64_t>(sms, items * tiles));
    prefix_parts = (size_t)(KVH * s.segments + s.grid) * s.R;
  }
  if (pl.own_kernel == kSpanSlots) {
    split_keys(max_length, (TG + slot_rows(TG) - 1) / slot_rows(TG) * B * KVH, 8 * (int64_t)sms, 128,
               &pl.own);
    own_parts = (size_t)pl.own.slots * rows;
  }
  const bool prefix_mma = pl.prefix_kernel == kSpanMma, own_mma = pl.own_kernel == kSpanMma;
  if (prefix_mma || own_mma) {  // one launch: the prefix's segments, then those of own contexts
    pl.nt = span_nt(prefix_mma ? all : TG);
    const int R = 8 * pl.nt;
    pdb::PartSet s{};
    s.kind = pdb::kPartUnits;
    s.R = R;
    int64_t units = 0, segments = 0;
    if (prefix_mma) {
      pl.prefix = s;
      pl.prefix.segments = (int)((all + R - 1) / R);
      segments = KVH * pl.prefix.segments;
      units = segments * ((P + 63) / 64 + pdb::kSpanOverhead);
    }
    if (own_mma) {
      pl.own = s;
      pl.own.segments = (int)((TG + R - 1) / R);
      pl.own.first = (int)segments;
      segments += B * KVH * pl.own.segments;
      units += B * KVH * pl.own.segments * ((max_length + 63) / 64 + pdb::kSpanOverhead);
    }
    const int grid = (int)std::min<int64_t>(kSpanCtasPerSm * (int64_t)(sms - beside_sms), units);
    pl.prefix.grid = prefix_mma ? grid : pl.prefix.grid;
    pl.own.grid = own_mma ? grid : pl.own.grid;
    own_parts = (size_t)(segments + grid) * R;
    span_segments = (size_t)segments;
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  pl.prefix_ml = take(prefix_parts * sizeof(float2));
  pl.prefix_o = take(prefix_parts * D * sizeof(float));
  pl.own_ml = take(own_parts * sizeof(float2));
  pl.own_o = take(own_parts * D * sizeof(float));
  pl.prefix_dir = take((size_t)(KVH * pl.prefix.segments) * sizeof(int2));
  pl.own_dir = take(span_segments * sizeof(int2));
  if (prefix_mma) {
    pl.prefix_ml = pl.own_ml;
    pl.prefix_o = pl.own_o;
    pl.prefix_dir = pl.own_dir;
  }
  pl.lse_off = take(scored ? (size_t)rows * sizeof(float) : 0);
  pl.logits_off = take(scored ? (size_t)rows * (size_t)max_length * sizeof(float) : 0);
  pl.total = at;
  return pl;
}

template <typename T, int DP, int RT>
cudaError_t launch_prefix_simt(int dev, const pdb::PrefixParams& p, bool prefix, cudaStream_t st) {
  using C = pdb::PrefixSimt<DP, RT>;
  auto* fn = &pdb::prefix_simt_kernel<T, DP, RT>;
  if (ctas_per_sm(dev, reinterpret_cast<const void*>(fn), C::SMEM, C::NT) <= 0)
    return cudaErrorInvalidConfiguration;
  const int64_t TG = (int64_t)p.T * p.G;
  const int prefix_tiles = prefix ? (int)((p.B * TG + RT - 1) / RT) : 0;
  const int own_tiles = prefix ? 0 : (int)((TG + RT - 1) / RT);
  const int64_t gx = prefix ? (int64_t)prefix_tiles * p.prefix.slots
                            : (int64_t)p.B * own_tiles * p.own.slots;
  return launch_pdl(fn, dim3((unsigned)gx, (unsigned)p.KVH), dim3(C::NT), C::SMEM, st, p,
                    prefix_tiles, own_tiles);
}
template <int D, int KW>
cudaError_t launch_prefix_tf32(int dev, const pdb::PrefixParams& p, bool prefix, cudaStream_t st) {
  using C = pdb::SpanTf32<D, KW>;
  auto* fn = &pdb::prefix_tf32_kernel<C>;
  if (ctas_per_sm(dev, reinterpret_cast<const void*>(fn), C::SMEM, C::NT) <= 0)
    return cudaErrorInvalidConfiguration;
  const int64_t TG = (int64_t)p.T * p.G;
  const int prefix_tiles = prefix ? (int)((p.B * TG + C::RT - 1) / C::RT) : 0;
  const int own_tiles = prefix ? 0 : (int)((TG + C::RT - 1) / C::RT);
  const int64_t gx = prefix ? (int64_t)prefix_tiles * p.prefix.slots
                            : (int64_t)p.B * own_tiles * p.own.slots;
  return launch_pdl(fn, dim3((unsigned)gx, (unsigned)p.KVH), dim3(C::NT), C::SMEM, st, p,
                    prefix_tiles, own_tiles);
}
template <int DP, int R>
cudaError_t launch_prefix_few(int dev, const pdb::PrefixParams& p, cudaStream_t st) {
  using C = pdb::PrefixFew<DP, R>;
  auto* fn = &pdb::prefix_few_kernel<DP, R>;
  if (ctas_per_sm(dev, reinterpret_cast<const void*>(fn), C::SMEM, C::NT) <= 0)
    return cudaErrorInvalidConfiguration;
  return launch_pdl(fn, dim3((unsigned)((int64_t)p.B * p.own.slots), (unsigned)p.KVH), dim3(C::NT),
                    C::SMEM, st, p);
}
template <typename T, int DP>
cudaError_t launch_prefix_simt_rows(int dev, const pdb::PrefixParams& p, bool prefix,
                                    cudaStream_t st) {
  const int rt = simt_rows((prefix ? p.B : 1) * (int64_t)p.T * p.G);
  if (rt == 8) return launch_prefix_simt<T, DP, 8>(dev, p, prefix, st);
  if (rt == 32) return launch_prefix_simt<T, DP, 32>(dev, p, prefix, st);
  return launch_prefix_simt<T, DP, 64>(dev, p, prefix, st);
}
template <int D>
cudaError_t launch_spans_fp32(int dev, const pdb::PrefixParams& p, bool prefix, cudaStream_t st) {
  const int64_t rows = (prefix ? p.B : 1) * (int64_t)p.T * p.G;
  if (!prefix && rows <= 4) return launch_prefix_few<D, 4>(dev, p, st);
  if (!prefix && rows <= 8) return launch_prefix_few<D, 8>(dev, p, st);
  const int rt = slot_rows(rows);
  if (rt == 16) return launch_prefix_tf32<D, 4>(dev, p, prefix, st);
  if (rt == 32) return launch_prefix_tf32<D, 2>(dev, p, prefix, st);
  return launch_prefix_tf32<D, 1>(dev, p, prefix, st);
}
// The spans of the prefix (or of own tokens) where key ranges are slots. `pieces`: FP32 with
// rows of 16-byte pieces and the kernels made for it (head_dim 64, 128) not ruled out.
cudaError_t launch_spans_slots(int dev, int dtype, const pdb::PrefixParams& p, bool prefix,
                               bool pieces, cudaStream_t st) {
  if (dtype == PDB_DTYPE_FLOAT16) {
    if (p.D <= 64) return launch_prefix_simt_rows<__half, 64>(dev, p, prefix, st);
    if (p.D <= 128) return launch_prefix_simt_rows<__half, 128>(dev, p, prefix, st);
    return launch_prefix_simt_rows<__half, 256>(dev, p, prefix, st);
  }
  if (pieces && p.D == 64) return launch_spans_fp32<64>(dev, p, prefix, st);
  if (pieces && p.D == 128) return launch_spans_fp32<128>(dev, p, prefix, st);
  if (p.D <= 64) return launch_prefix_simt_rows<float, 64>(dev, p, prefix, st);
  if (p.D <= 128) return launch_prefix_simt_rows<float, 128>(dev, p, prefix, st);
  return launch_prefix_simt_rows<float, 256>(dev, p, prefix, st);
}

// ROWS 8, 16, 32 (NT tiles of 8 per warp, RW row groups).
template <int D, int NT, int RW>
cudaError_t launch_span_mma(int dev, const pdb::PrefixParams& p, const pdb::SpanSet& ss, int grid,
                            cudaStream_t st, const CUtensorMap& kmap, const CUtensorMap& vmap) {
  using C = pdb::SpanMma<D, NT, RW, (D == 128 && RW == 2) ? 2 : 3>;
  auto* fn = &pdb::prefix_span_kernel<C>;
  if (ctas_per_sm(dev, reinterpret_cast<const void*>(fn), C::SMEM, C::THREADS) <= 0)
    return cudaErrorInvalidConfiguration;
  return launch_pdl(fn, dim3((unsigned)grid), dim3(C::THREADS), C::SMEM, st, p, ss, kmap, vmap);
}
cudaError_t launch_spans_mma(int dev, const pdb::PrefixParams& p, const PrefixPlan& pl,
                             cudaStream_t st, const CUtensorMap& kmap, const CUtensorMap& vmap) {
  pdb::SpanSet ss{};
  ss.has_prefix = pl.prefix_kernel == kSpanMma ? 1 : 0;
  ss.nseq = pl.own_kernel == kSpanMma ? p.B : 0;
  ss.part = ss.nseq ? p.own : p.prefix;
  ss.prefix_segments = ss.has_prefix ? p.prefix.segments : 0;
  ss.beside = p.beside;
  const int nt = pl.nt, grid = ss.part.grid;
  if (p.D == 64) {
    if (nt == 1) return launch_span_mma<64, 1, 1>(dev, p, ss, grid, st, kmap, vmap);
    if (nt == 2) return launch_span_mma<64, 2, 1>(dev, p, ss, grid, st, kmap, vmap);
    return launch_span_mma<64, 2, 2>(dev, p, ss, grid, st, kmap, vmap);
  }
  if (nt == 1) return launch_span_mma<128, 1, 1>(dev, p, ss, grid, st, kmap, vmap);
  if (nt == 2) return launch_span_mma<128, 2, 1>(dev, p, ss, grid, st, kmap, vmap);
  return launch_span_mma<128, 2, 2>(dev, p, ss, grid, st, kmap, vmap);
}

// Pool [N, bs, KVH, D] as [64 columns, N * bs rows, D / 64 halves, KVH]; box = one
// 16-token unit of one kv head, all its columns, half by half; 128-byte swizzle.
bool encode_unit_map(CUtensorMap* m, const void* pool, int64_t N, int64_t bs, int64_t KVH,
                     int64_t D) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[4] = {64, (cuuint64_t)(N * bs), (cuuint64_t)(D / 64), (cuuint64_t)KVH};
  const cuuint64_t strides[3] = {(cuuint64_t)(KVH * D * 2), 128, (cuuint64_t)(D * 2)};
  const cuuint32_t box[4] = {64, (cuuint32_t)pdb::kUnitTokens, (cuuint32_t)(D / 64), 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pool), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query tiles of the tcgen05 kernel: box {64 columns, G heads, `tokens` tokens}.
bool encode_group_map(CUtensorMap* m, const void* q, int64_t R, int64_t heads, int64_t D, int G,
                      int tokens) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)R};
  const cuuint64_t strides[2] = {(cuuint64_t)(D * 2), (cuuint64_t)(heads * D * 2)};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)tokens};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <int D>
cudaError_t launch_prefix_tc(int dev, const pdb::PrefixParams& p, int splits, cudaStream_t st,
                             const CUtensorMap& kmap, const CUtensorMap& vmap) {
  using C = pdb::PrefixTc<D>;
  auto* fn = &pdb::prefix_tc_kernel<D>;
  if (ctas_per_sm(dev, reinterpret_cast<const void*>(fn), C::SMEM, C::THREADS) <= 0)
    return cudaErrorInvalidConfiguration;
  pdb::PrefixTcParams t{};
  t.table = p.prefix_table;
  t.ml = p.prefix.ml;
  t.o = p.prefix.o;
  t.num_blocks = p.num_blocks;
  t.tokens = p.B * p.T;
  t.H = p.H; t.KVH = p.KVH; t.G = p.G;
  t.per_tile = p.prefix.half;
  t.pairs = p.prefix.segments;
  t.key_tiles = (p.prefix_length + C::BN - 1) / C::BN;
  t.splits = splits;
  t.dir = p.prefix.dir;
  t.prefix_length = p.prefix_length;
  t.block_size = p.block_size; t.bs_shift = p.bs_shift;
  t.scale_log2 = p.scale_log2;
  CUtensorMap qmap;
  if (!encode_group_map(&qmap, p.q, t.tokens, p.H, D, p.G, t.per_tile)) return cudaErrorInvalidValue;
  return launch_pdl(fn, dim3((unsigned)p.prefix.grid), dim3(C::THREADS), C::SMEM, st, t, qmap, kmap,
                    vmap);
}

// Whether the tensor-core kernels take this shape (pointers aside).
bool prefix_tensor_cores(int64_t D, int64_t num_blocks, int64_t block_size, int dtype) {
  return dtype == PDB_DTYPE_FLOAT16 && (D == 64 || D == 128) &&
         block_size % pdb::kUnitTokens == 0 && num_blocks * block_size <= INT32_MAX &&
         tensor_map_encoder() != nullptr;
}

// Sizes that every kernel's 32-bit indices can hold.
bool prefix_sizes_ok(int64_t B, int64_t T, int64_t H, int64_t D, int64_t KVH, int64_t P,
                     int64_t max_length) {
  const int64_t lim = int64_t(1) << 30;
  return B <= 65535 && T <= 4096 && H <= 4096 && KVH <= 65535 && P <= lim && max_length <= lim &&
         B * T * H * D < (int64_t(1) << 40) && B * T * H < (int64_t(1) << 30);
}

}  // namespace

extern "C" {

size_t pdb_shared_prefix_attention_workspace_size(int64_t batch, int64_t tokens, int64_t heads,
                                                  int64_t kv_heads, int64_t head_dim,
                                                  int64_t prefix_length, int64_t max_length,
                                                  int dtype, int with_scores) {
  if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
      heads % kv_heads || prefix_length < 0 || max_length < 0 ||
      !prefix_sizes_ok(batch, tokens, heads, head_dim, kv_heads, prefix_length, max_length))
    return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  // the pool is not known here: cover every kernel that a call may select
  const int sms = sm_count(dev);
  size_t need = 0;
  const int impls[4] = {PDB_PREFIX_AUTO, PDB_PREFIX_SIMT, PDB_PREFIX_MMA, PDB_PREFIX_TCGEN05};
  for (const int impl : impls) {
    const size_t n =
        prefix_plan(sms, batch, tokens, heads, kv_heads, head_dim, prefix_length, max_length,
                    with_scores != 0, prefix_tensor_cores(head_dim, 1, 16, dtype), impl).total;
    if (n > need) need = n;
  }
  return need;
}

int pdb_shared_prefix_attention_impl(
    const void* q, const void* k_pool, const void* v_pool, const int32_t* prefix_table,
    int64_t prefix_pages, int64_t prefix_length, const int32_t* tables, const int32_t* lengths,
    const int32_t* counts, const float* scores, float* scores_out, int64_t scores_width, void* out,
    int64_t batch, int64_t tokens, int64_t heads, int64_t head_dim, int64_t num_blocks,
    int64_t block_size, int64_t kv_heads, int64_t table_width, int64_t max_length, int dtype,
    void* workspace, size_t workspace_bytes, void* stream, int impl) {
  if (!(batch > 0 && tokens > 0 && heads > 0 && head_dim > 0 && head_dim <= 256))
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid query shape");
  if (!(num_blocks > 0 && block_size > 0 && kv_heads > 0))
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid cache shape");
  if (heads % kv_heads)
    return fail(PDB_ERR_INVALID_ARGUMENT, "query heads must be a multiple of KV heads");
  if (dtype != PDB_DTYPE_FLOAT32 && dtype != PDB_DTYPE_FLOAT16)
    return fail(PDB_ERR_INVALID_ARGUMENT, "use FP32 or FP16");
  if (table_width < 0 || prefix_pages < 0)
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid block tables");
  if (block_size > (1 << 20) || table_width > INT32_MAX || prefix_pages > INT32_MAX ||
      num_blocks > INT64_MAX / (block_size * kv_heads * head_dim * 4) ||
      !prefix_sizes_ok(batch, tokens, heads, head_dim, kv_heads, prefix_length, max_length))
    return fail(PDB_ERR_INVALID_ARGUMENT, "shape too large");
  if (prefix_length < 0 || prefix_pages * block_size < prefix_length)
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid prefix length");
  if (max_length < 0 || table_width * block_size < max_length)
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid context bound");
  if ((scores == nullptr) != (scores_out == nullptr))
    return fail(PDB_ERR_INVALID_ARGUMENT, "give both scores and their output");
  if (scores && scores_width < max_length)
    return fail(PDB_ERR_INVALID_ARGUMENT, "scores must hold max_length tokens");
  if (scores && (scores_width > INT32_MAX ||
                 (scores_width + 1023) / 1024 > INT32_MAX / (batch * kv_heads)))
    return fail(PDB_ERR_INVALID_ARGUMENT, "shape too large");
  if (impl < PDB_PREFIX_AUTO || impl > PDB_PREFIX_TCGEN05)
    return fail(PDB_ERR_INVALID_ARGUMENT, "unknown kernel selection");
  if (!q || !k_pool || !v_pool || !lengths || !out || (prefix_length > 0 && !prefix_table) ||
      (max_length > 0 && !tables))
    return fail(PDB_ERR_INVALID_ARGUMENT, "null tensor pointer");
  int dev = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  const bool aligned = aligned16(q) && aligned16(k_pool) && aligned16(v_pool);
  const bool tensor_cores =
      prefix_tensor_cores(head_dim, num_blocks, block_size, dtype) && aligned;
  const bool pieces = aligned && impl != PDB_PREFIX_SIMT;
  if (impl > PDB_PREFIX_SIMT && !tensor_cores)
    return fail(PDB_ERR_INVALID_ARGUMENT, "tensor-core kernels do not support this shape/alignment");
  const PrefixPlan pl = prefix_plan(sm_count(dev), batch, tokens, heads, kv_heads, head_dim,
                                    prefix_length, max_length, scores != nullptr, tensor_cores, impl);
  if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(PDB_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  if (pl.total && (!workspace || workspace_bytes < pl.total))
    return fail(PDB_ERR_WORKSPACE,
                "workspace too small: need " + std::to_string(pl.total) + " bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* wb = static_cast<unsigned char*>(workspace);
  pdb::PrefixParams p{};
  p.q = q; p.k_pool = k_pool; p.v_pool = v_pool;
  p.prefix_table = prefix_table; p.tables = tables; p.lengths = lengths; p.counts = counts;
  p.out = out;
  p.prefix = pl.prefix;
  p.prefix.ml = reinterpret_cast<float2*>(wb + pl.prefix_ml);
  p.prefix.o = reinterpret_cast<float*>(wb + pl.prefix_o);
  p.own = pl.own;
  p.own.ml = reinterpret_cast<float2*>(wb + pl.own_ml);
  p.own.o = reinterpret_cast<float*>(wb + pl.own_o);
  p.prefix.dir = reinterpret_cast<int2*>(wb + pl.prefix_dir);
  p.own.dir = reinterpret_cast<int2*>(wb + pl.own_dir);
  if (scores) {
    p.lse = reinterpret_cast<float*>(wb + pl.lse_off);
    p.logits = reinterpret_cast<float*>(wb + pl.logits_off);
  }
  p.scores = scores; p.scores_out = scores_out;
  p.num_blocks = num_blocks; p.rows = batch * tokens * heads;
  p.logits_width = max_length; p.scores_width = scores_width;
  p.B = (int)batch; p.T = (int)tokens; p.H = (int)heads; p.KVH = (int)kv_heads;
  p.G = (int)(heads / kv_heads); p.D = (int)head_dim;
  p.block_size = (int)block_size; p.bs_shift = page_shift(block_size);
  p.table_width = (int)table_width;
  p.prefix_length = (int)prefix_length; p.max_length = (int)max_length;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
  p.beside = (pl.prefix_kernel == kSpanTc || pl.prefix_kernel == kSpanSlots) && pl.own_kernel;
  CUtensorMap kmap, vmap, kunits, vunits;  // boxes of the tcgen05 kernel, of the mma.sync kernel
  const bool tc = pl.prefix_kernel == kSpanTc;
  const bool mma = pl.prefix_kernel == kSpanMma || pl.own_kernel == kSpanMma;
  if ((tc && !(encode_pool_map(&kmap, k_pool, num_blocks, block_size, kv_heads, head_dim) &&
               encode_pool_map(&vmap, v_pool, num_blocks, block_size, kv_heads, head_dim))) ||
      (mma && !(encode_unit_map(&kunits, k_pool, num_blocks, block_size, kv_heads, head_dim) &&
                encode_unit_map(&vunits, v_pool, num_blocks, block_size, kv_heads, head_dim))))
    return fail(PDB_ERR_CUDA, "cuTensorMapEncodeTiled failed for the KV pools");
  cudaError_t e = cudaSuccess;
  if (pl.prefix_kernel == kSpanTc)
    e = head_dim == 64 ? launch_prefix_tc<64>(dev, p, pl.splits, st, kmap, vmap)
                       : launch_prefix_tc<128>(dev, p, pl.splits, st, kmap, vmap);
  else if (pl.prefix_kernel == kSpanSlots)
    e = launch_spans_slots(dev, dtype, p, true, pieces, st);
  if (e == cudaSuccess && mma)
    e = launch_spans_mma(dev, p, pl, st, kunits, vunits);
  else if (e == cudaSuccess && pl.own_kernel == kSpanSlots)
    e = launch_spans_slots(dev, dtype, p, false, pieces, st);
  if (e == cudaSuccess) {
    auto join = [&](auto* fn, int lanes) {
      const int threads = std::min(256, (p.H * lanes + 31) / 32 * 32);
      const dim3 grid((unsigned)(batch * tokens),
                      (unsigned)((p.H * lanes + threads - 1) / threads));
      return launch_pdl(fn, grid, dim3((unsigned)threads), 0, st, p);
    };
    const bool vec = head_dim % 4 == 0 && head_dim <= 128;
    if (dtype == PDB_DTYPE_FLOAT16)
      e = !vec             ? join(pdb::prefix_join_kernel<__half, 32, false>, 32)
          : head_dim <= 64 ? join(pdb::prefix_join_kernel<__half, 16, true>, 16)
                           : join(pdb::prefix_join_kernel<__half, 32, true>, 32);
    else
      e = !vec             ? join(pdb::prefix_join_kernel<float, 32, false>, 32)
          : head_dim <= 64 ? join(pdb::prefix_join_kernel<float, 16, true>, 16)
                           : join(pdb::prefix_join_kernel<float, 32, true>, 32);
  }
  if (e == cudaSuccess && scores && scores_width > 0)
    e = launch_pdl(pdb::prefix_scores_kernel,
                   dim3((unsigned)((scores_width + 1023) / 1024 * p.B * p.KVH)), dim3(256), 0, st,
                   p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "shared prefix attention launch");
  return PDB_OK;
}

int pdb_shared_prefix_attention(
    const void* q, const void* k_pool, const void* v_pool, const int32_t* prefix_table,
    int64_t prefix_pages, int64_t prefix_length, const int32_t* tables, const int32_t* lengths,
    const int32_t* counts, const float* scores, float* scores_out, int64_t scores_width, void* out,
    int64_t batch, int64_t tokens, int64_t heads, int64_t head_dim, int64_t num_blocks,
    int64_t block_size, int64_t kv_heads, int64_t table_width, int64_t max_length, int dtype,
    void* workspace, size_t workspace_bytes, void* stream) {
  return pdb_shared_prefix_attention_impl(
      q, k_pool, v_pool, prefix_table, prefix_pages, prefix_length, tables, lengths, counts,
      scores, scores_out, scores_width, out, batch, tokens, heads, head_dim, num_blocks,
      block_size, kv_heads, table_width, max_length, dtype, workspace, workspace_bytes, stream,
      PDB_PREFIX_AUTO);
}

int pdb_verify_drafts(const int64_t* draft_tokens, const void* target_probs,
                      const void* draft_probs, const float* accept_uniforms,
                      const float* sample_uniforms, const int32_t* draft_lengths, int64_t* tokens,
                      int32_t* counts, int64_t batch, int64_t drafts, int64_t vocab, int dtype,
                      void* stream) {
  if (!(batch > 0 && drafts > 0 && vocab > 0))
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid probabilities shape");
  if (dtype != PDB_DTYPE_FLOAT32 && dtype != PDB_DTYPE_FLOAT16)
    return fail(PDB_ERR_INVALID_ARGUMENT, "use FP32 or FP16");
  // 2^22 weights of at most 2^40 each stay below 2^63
  if (vocab > (int64_t(1) << 22) || drafts > (1 << 20) || batch > (1 << 27))
    return fail(PDB_ERR_INVALID_ARGUMENT, "shape too large");
  if (!draft_tokens || !target_probs || !accept_uniforms || !sample_uniforms || !tokens || !counts)
    return fail(PDB_ERR_INVALID_ARGUMENT, "null tensor pointer");
  pdb::VerifyParams p{};
  p.draft_tokens = draft_tokens; p.target = target_probs; p.draft = draft_probs;
  p.accept_uniforms = accept_uniforms; p.sample_uniforms = sample_uniforms;
  p.draft_lengths = draft_lengths; p.tokens = tokens; p.counts = counts;
  p.V = vocab; p.B = (int)batch; p.T = (int)drafts;
  int dev = 0;
  const int rc = current_device(&dev);
  if (rc) return rc;
  // CTAs per sequence: up to four per SM in all, each with 2048 entries at least (256
  // rows of 100003: 41 us with 2 CTAs, 58 with 1, 45 with 4; one row of 49152: 7.0 us
  // with 8, 15.8 with 1)
  int C = 1;
  while (C < pdb::kVerifyMaxCluster && batch * C * 2 <= 4 * (int64_t)sm_count(dev) &&
         vocab / (2 * C) >= 2048)
    C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * C));
  cfg.blockDim = dim3(pdb::kVerifyThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = dtype == PDB_DTYPE_FLOAT16
                      ? cudaLaunchKernelEx(&cfg, pdb::verify_kernel<__half>, p)
                      : cudaLaunchKernelEx(&cfg, pdb::verify_kernel<float>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "verify drafts launch");
  return PDB_OK;
}

int pdb_evict_tokens(void* k_pool, void* v_pool, const float* scores, int64_t scores_width,
                     const int32_t* tables, const int32_t* lengths, const int32_t* new_tables,
                     int32_t* kept, int32_t* new_lengths, float* new_scores, int64_t batch,
                     int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t kv_heads,
                     int64_t table_width, int64_t new_table_width, int64_t budget, int64_t recent,
                     int dtype, void* stream) {
  if (!(batch > 0 && num_blocks > 0 && block_size > 0 && kv_heads > 0 && head_dim > 0))
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid cache shape");
  if (dtype != PDB_DTYPE_FLOAT32 && dtype != PDB_DTYPE_FLOAT16)
    return fail(PDB_ERR_INVALID_ARGUMENT, "use FP32 or FP16");
  if (scores_width <= 0) return fail(PDB_ERR_INVALID_ARGUMENT, "invalid scores");
  if (table_width <= 0 || new_table_width <= 0)
    return fail(PDB_ERR_INVALID_ARGUMENT, "invalid block tables");
  if (batch > 65535 || kv_heads > 65535 || head_dim > 65536 || block_size > (1 << 20) ||
      batch * kv_heads > INT32_MAX || kv_heads * head_dim > (1 << 22) ||
      table_width > INT32_MAX || new_table_width > INT32_MAX || scores_width > (1 << 30) ||
      num_blocks > INT64_MAX / (block_size * kv_heads * head_dim * 4))
    return fail(PDB_ERR_INVALID_ARGUMENT, "shape too large");
  if (budget <= 0 || budget > (1 << 30)) return fail(PDB_ERR_INVALID_ARGUMENT, "invalid budget");
  if (recent < 0 || recent > budget)
    return fail(PDB_ERR_INVALID_ARGUMENT, "recent tokens must fit the budget");
  const int64_t most = budget < scores_width ? budget : scores_width;
  if (new_table_width * block_size < (most < table_width * block_size ? most
                                                                      : table_width * block_size))
    return fail(PDB_ERR_INVALID_ARGUMENT, "new tables must hold the budget");
  if (!k_pool || !v_pool || !scores || !tables || !lengths || !new_tables || !kept ||
      !new_lengths || !new_scores)
    return fail(PDB_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (new_scores == scores)
    return fail(PDB_ERR_INVALID_ARGUMENT, "new scores must not overwrite the scores");
  pdb::EvictParams p{};
  p.k_pool = k_pool; p.v_pool = v_pool; p.scores = scores;
  p.tables = tables; p.lengths = lengths; p.new_tables = new_tables;
  p.kept = kept; p.new_lengths = new_lengths; p.new_scores = new_scores;
  p.num_blocks = num_blocks; p.S = scores_width;
  p.B = (int)batch; p.KVH = (int)kv_heads; p.W = (int)table_width; p.W2 = (int)new_table_width;
  p.block_size = (int)block_size; p.bs_shift = page_shift(block_size);
  p.budget = (int)budget; p.recent = (int)recent;
  const int esize = dtype == PDB_DTYPE_FLOAT16 ? 2 : 4;
  const bool wide = head_dim * esize % 16 == 0 && aligned16(k_pool) && aligned16(v_pool);
  p.row_pieces = (int)(wide ? head_dim * esize / 16 : head_dim);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 sel((unsigned)(batch * kv_heads));
  // Where a head's rows are few its selecting CTA copies them too (3 heads of 256 rows of
  // 128 bytes: 7.9 us on the device against 7.2 in two launches, but 2.4 us less of the
  // host's time per call, which is what bounds calls of this size); else a second kernel
  // spreads them over more CTAs (48 x 8 heads of 1024 rows of 256 bytes: 96 us against
  // 100, 8 heads of as many rows several times).
  const bool own_rows = most * head_dim * esize <= (64 << 10);
  cudaError_t e = cudaSuccess;
  auto select = [&](auto piece) {
    using P = decltype(piece);
    using Q = typename std::conditional<std::is_same<P, char>::value, void, P>::type;
    // scores per thread that fit one round of the CTA; longer caches take rounds
    e = scores_width <= 4 * pdb::kEvictThreads
            ? launch_pdl(pdb::evict_select_kernel<4, Q>, sel, dim3(pdb::kEvictThreads), 0, st, p)
            : launch_pdl(pdb::evict_select_kernel<16, Q>, sel, dim3(pdb::kEvictThreads), 0, st, p);
  };
  if (!own_rows) select(char());  // no piece: selection only
  else if (wide) select(uint4());
  else if (esize == 2) select(uint16_t());
  else select(uint32_t());
  if (e == cudaSuccess && !own_rows) {
    const dim3 grid((unsigned)((most + pdb::kEvictCells - 1) / pdb::kEvictCells), (unsigned)batch,
                    (unsigned)((kv_heads + pdb::kEvictHeads - 1) / pdb::kEvictHeads));
    if (wide)
      e = launch_pdl(pdb::evict_move_kernel<uint4>, grid, dim3(256), 0, st, p);
    else if (esize == 2)
      e = launch_pdl(pdb::evict_move_kernel<uint16_t>, grid, dim3(256), 0, st, p);
    else
      e = launch_pdl(pdb::evict_move_kernel<uint32_t>, grid, dim3(256), 0, st, p);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "evict tokens launch");
  return PDB_OK;
}

}  // extern "C"
