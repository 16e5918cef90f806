// C entry points of the shared-prefix attention, the verification of drafted
// tokens and the cache eviction: argument checks, kernel selection, workspace
// layout and launches. Included by paged_decode.cu, whose helpers it uses.
#pragma once

#include "shared_prefix.cuh"
#include "verify.cuh"
#include "evict.cuh"

namespace {

int page_shift(int64_t bs) {
  return (bs & (bs - 1)) == 0 ? __builtin_ctzll((unsigned long long)bs) : -1;
}

// ---- shared-prefix attention -------------------------------------------------
struct PrefixPlan {
  int prefix_slots, prefix_chunk, own_slots, own_chunk;
  size_t ml_off, o_off, lse_off, logits_off, total;
};

// Splits `keys` into ranges of a multiple of 64 keys, no shorter than `least`,
// so that `tiles` CTAs per range reach `want` CTAs where the keys allow it.
void split_keys(int64_t keys, int64_t tiles, int64_t want, int64_t least, int* slots, int* chunk) {
  if (keys <= 0) {
    *slots = 0;
    *chunk = 64;
    return;
  }
  int64_t s = (want + tiles - 1) / tiles;
  const int64_t most = (keys + least - 1) / least;
  if (s > most) s = most;
  if (s < 1) s = 1;
  int64_t c = (keys + s - 1) / s;
  c = (c + 63) / 64 * 64;
  *chunk = (int)c;
  *slots = (int)((keys + c - 1) / c);
}

constexpr int kPrefixSimtRows = 32;
int simt_rows(int64_t rows) { return rows <= 8 ? 8 : kPrefixSimtRows; }

PrefixPlan prefix_plan(int64_t B, int64_t T, int64_t H, int64_t KVH, int64_t D, int64_t P,
                       int64_t max_length, bool scored) {
  PrefixPlan pl{};
  const int64_t TG = T * (H / KVH), rows = B * T * H;
  const int64_t pt = (B * TG + simt_rows(B * TG) - 1) / simt_rows(B * TG);
  const int64_t ot = (TG + simt_rows(TG) - 1) / simt_rows(TG);
  split_keys(P, pt * KVH, 4 * 148, 64, &pl.prefix_slots, &pl.prefix_chunk);
  split_keys(max_length, ot * B * KVH, 8 * 148, 128, &pl.own_slots, &pl.own_chunk);
  const size_t slots = (size_t)pl.prefix_slots + pl.own_slots;
  pl.ml_off = 0;
  pl.o_off = align256(slots * rows * sizeof(float2));
  pl.lse_off = pl.o_off + align256(slots * rows * D * sizeof(float));
  pl.logits_off = pl.lse_off + (scored ? align256((size_t)rows * sizeof(float)) : 0);
  pl.total = pl.logits_off +
             (scored ? align256((size_t)rows * (size_t)max_length * sizeof(float)) : 0);
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
  const int64_t gx = prefix ? (int64_t)prefix_tiles * p.prefix_slots
                            : (int64_t)p.B * own_tiles * p.own_slots;
  return launch_pdl(fn, dim3((unsigned)gx, (unsigned)p.KVH), dim3(C::NT), C::SMEM, st, p,
                    prefix_tiles, own_tiles);
}
template <typename T, int DP>
cudaError_t launch_prefix_simt_rows(int dev, const pdb::PrefixParams& p, bool prefix,
                                    cudaStream_t st) {
  const int64_t rows = (prefix ? p.B : 1) * (int64_t)p.T * p.G;
  if (simt_rows(rows) == 8) return launch_prefix_simt<T, DP, 8>(dev, p, prefix, st);
  return launch_prefix_simt<T, DP, kPrefixSimtRows>(dev, p, prefix, st);
}
// The spans of the prefix (or of own tokens) on the FP32 pipes.
cudaError_t launch_spans_simt(int dev, int dtype, const pdb::PrefixParams& p, bool prefix,
                              cudaStream_t st) {
  if (dtype == PDB_DTYPE_FLOAT16) {
    if (p.D <= 64) return launch_prefix_simt_rows<__half, 64>(dev, p, prefix, st);
    if (p.D <= 128) return launch_prefix_simt_rows<__half, 128>(dev, p, prefix, st);
    return launch_prefix_simt_rows<__half, 256>(dev, p, prefix, st);
  }
  if (p.D <= 64) return launch_prefix_simt_rows<float, 64>(dev, p, prefix, st);
  if (p.D <= 128) return launch_prefix_simt_rows<float, 128>(dev, p, prefix, st);
  return launch_prefix_simt_rows<float, 256>(dev, p, prefix, st);
}

// Sizes that every kernel's 32-bit indices can hold.
bool prefix_sizes_ok(int64_t B, int64_t T, int64_t H, int64_t D, int64_t KVH, int64_t P,
                     int64_t max_length) {
  const int64_t lim = int64_t(1) << 30;
  return B <= 65535 && T <= 4096 && H <= 4096 && KVH <= 65535 && P <= lim && max_length <= lim &&
         B * T * H * D < (int64_t(1) << 40) && B * T * H < (int64_t(1) << 31);
}

}  // namespace

extern "C" {

size_t pdb_shared_prefix_attention_workspace_size(int64_t batch, int64_t tokens, int64_t heads,
                                                  int64_t kv_heads, int64_t head_dim,
                                                  int64_t prefix_length, int64_t max_length,
                                                  int dtype, int with_scores) {
  (void)dtype;
  if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
      heads % kv_heads || prefix_length < 0 || max_length < 0 ||
      !prefix_sizes_ok(batch, tokens, heads, head_dim, kv_heads, prefix_length, max_length))
    return 0;
  return prefix_plan(batch, tokens, heads, kv_heads, head_dim, prefix_length, max_length,
                     with_scores != 0)
      .total;
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
  if (scores && scores_width > INT32_MAX) return fail(PDB_ERR_INVALID_ARGUMENT, "shape too large");
  if (impl < PDB_PREFIX_AUTO || impl > PDB_PREFIX_SIMT)
    return fail(PDB_ERR_INVALID_ARGUMENT, "unknown kernel selection");
  if (!q || !k_pool || !v_pool || !lengths || !out || (prefix_length > 0 && !prefix_table) ||
      (max_length > 0 && !tables))
    return fail(PDB_ERR_INVALID_ARGUMENT, "null tensor pointer");
  const PrefixPlan pl = prefix_plan(batch, tokens, heads, kv_heads, head_dim, prefix_length,
                                    max_length, scores != nullptr);
  if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(PDB_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  if (pl.total && (!workspace || workspace_bytes < pl.total))
    return fail(PDB_ERR_WORKSPACE,
                "workspace too small: need " + std::to_string(pl.total) + " bytes");
  int dev = 0;
  int rc = current_device(&dev);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* wb = static_cast<unsigned char*>(workspace);
  pdb::PrefixParams p{};
  p.q = q; p.k_pool = k_pool; p.v_pool = v_pool;
  p.prefix_table = prefix_table; p.tables = tables; p.lengths = lengths; p.counts = counts;
  p.out = out;
  p.ml = reinterpret_cast<float2*>(wb + pl.ml_off);
  p.o = reinterpret_cast<float*>(wb + pl.o_off);
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
  p.prefix_slots = pl.prefix_slots; p.prefix_chunk = pl.prefix_chunk;
  p.own_slots = pl.own_slots; p.own_chunk = pl.own_chunk;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
  cudaError_t e = cudaSuccess;
  if (p.prefix_slots) e = launch_spans_simt(dev, dtype, p, true, st);
  if (e == cudaSuccess && p.own_slots) e = launch_spans_simt(dev, dtype, p, false, st);
  if (e == cudaSuccess) {
    const dim3 grid((unsigned)((p.rows + 7) / 8));
    e = dtype == PDB_DTYPE_FLOAT16
            ? launch_pdl(pdb::prefix_join_kernel<__half>, grid, dim3(256), 0, st, p)
            : launch_pdl(pdb::prefix_join_kernel<float>, grid, dim3(256), 0, st, p);
  }
  if (e == cudaSuccess && scores && scores_width > 0)
    e = launch_pdl(pdb::prefix_scores_kernel,
                   dim3((unsigned)((scores_width + 255) / 256), (unsigned)(p.B * p.KVH)),
                   dim3(256), 0, st, p);
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
  // CTAs per sequence: enough for two per SM, but at least 2048 entries each
  int C = 1;
  while (C < pdb::kVerifyMaxCluster && batch * C < 2 * (int64_t)sm_count(dev) &&
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
  // scores per thread that fit one round of the CTA; longer caches take rounds
  cudaError_t e = scores_width <= 4 * pdb::kEvictThreads
                      ? launch_pdl(pdb::evict_select_kernel<4>, sel, dim3(pdb::kEvictThreads), 0, st, p)
                      : launch_pdl(pdb::evict_select_kernel<16>, sel, dim3(pdb::kEvictThreads), 0, st, p);
  if (e == cudaSuccess) {
    const dim3 grid((unsigned)((most + pdb::kEvictCells - 1) / pdb::kEvictCells), (unsigned)batch);
    if (wide)
      e = launch_pdl(pdb::evict_move_kernel<uint4>, grid, dim3(256), 0, st, p);
    else if (esize == 2)
      e = launch_pdl(pdb::evict_move_kernel<__half>, grid, dim3(256), 0, st, p);
    else
      e = launch_pdl(pdb::evict_move_kernel<float>, grid, dim3(256), 0, st, p);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "evict tokens launch");
  return PDB_OK;
}

}  // extern "C"
