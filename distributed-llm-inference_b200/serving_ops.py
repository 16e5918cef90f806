"""Operators of speculative serving over the C ABI.

``shared_prefix_attention`` scores one or more (drafted) tokens per sequence
against a prefix that the whole batch shares and each sequence's own pages,
optionally accumulating the attention weight that own tokens get;
``verify_drafts`` accepts drafted tokens against the target's probabilities;
``evict_tokens`` keeps a cache under a budget by those accumulated weights. The
reference has none of them: it decodes one token per step over each sequence's
whole context and keeps every token until the request ends. Checks, errors
(RuntimeError), streams and workspaces are those of ``ops``.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .ops import _DTYPES, _DeviceGuard, _check, _stream_ptr, workspace


def _check_same_device(first: torch.Tensor, *others) -> None:
    for t in (first, *others):
        if t is not None:
            _check(t.device == first.device, "all tensors must be on the same GPU")
            _check(t.is_contiguous(), "all tensors must be contiguous")


@functools.lru_cache(maxsize=1024)
def _prefix_workspace(device, B, T, H, KVH, D, prefix, longest, dt, scored) -> int:
    return _lib.load().pdb_shared_prefix_attention_workspace_size(B, T, H, KVH, D, prefix, longest,
                                                                  dt, scored)


def shared_prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            prefix_table: torch.Tensor, prefix_length: int, tables: torch.Tensor,
                            lengths: torch.Tensor, max_length: int, *,
                            counts: torch.Tensor | None = None,
                            scores: torch.Tensor | None = None,
                            scores_out: torch.Tensor | None = None,
                            out: torch.Tensor | None = None, impl: int = _lib.PREFIX_AUTO):
    """Attention of a batch that shares a prefix, the prefix read once for all.

    q [B, T, H, D] (or [B, H, D], one token per sequence); k, v
    [blocks, block_size, KVH, D]; ``prefix_table`` int32 [pages] whose first
    ``prefix_length`` tokens every query token sees; tables int32 [B, W] and
    lengths int32 [B] describe each sequence's own tokens, the T new ones
    included (lengths <= max_length). With ``counts`` int32 [B] only the first
    counts[b] query tokens are real: token t is own token
    lengths[b] - counts[b] + t and sees own tokens up to itself. Rows that are
    not real, or see nothing, are zeros. Returns q's shape and dtype
    (FP32 or FP16, head_dim <= 256).

    ``scores`` fp32 [B, KVH, S] (S >= max_length) adds up the softmax weight
    that each own token got, over the query tokens and the heads of its kv
    head: into ``scores_out`` (default: in place). Returns (out, scores) then.
    Asynchronous on the current stream; `impl` pins the kernels.
    """
    _check(q.is_cuda, "query must be on CUDA")
    _check_same_device(q, k, v, prefix_table, tables, lengths, counts, scores, scores_out)
    _check(q.dim() in (3, 4) and k.dim() == 4 and k.shape == v.shape, "invalid Q/K/V shapes")
    if q.dim() == 4:
        B, T, H, D = q.shape
    else:
        (B, H, D), T = q.shape, 1
    N, bs, KVH, Dk = k.shape
    _check(B > 0 and T > 0 and H > 0 and 0 < D <= 256, "invalid query shape")
    _check(N > 0 and bs > 0 and KVH > 0 and Dk == D, "invalid cache shape")
    _check(H % KVH == 0, "query heads must be a multiple of KV heads")
    _check(q.dtype in _DTYPES, "use FP32 or FP16")
    _check(k.dtype == q.dtype and v.dtype == q.dtype, "dtype mismatch")
    _check(tables.dtype == torch.int32 and lengths.dtype == torch.int32
           and prefix_table.dtype == torch.int32, "metadata must be int32")
    _check(tables.dim() == 2 and tables.size(0) == B and prefix_table.dim() == 1,
           "invalid block tables")
    _check(lengths.dim() == 1 and lengths.size(0) == B, "invalid lengths")
    if counts is not None:
        _check(counts.dtype == torch.int32 and counts.shape == (B,), "invalid token counts")
    prefix_length, max_length = int(prefix_length), int(max_length)
    _check(0 <= prefix_length <= prefix_table.size(0) * bs, "invalid prefix length")
    _check(0 <= max_length <= tables.size(1) * bs, "invalid context bound")
    width = 0
    if scores is not None:
        _check(scores.dtype == torch.float32 and scores.dim() == 3
               and scores.shape[:2] == (B, KVH), "scores must be fp32 [batch, kv_heads, tokens]")
        width = scores.size(2)
        _check(width >= max_length, "scores must hold max_length tokens")
        if scores_out is None:
            scores_out = scores
        _check(scores_out.shape == scores.shape and scores_out.dtype == torch.float32,
               "invalid scores output")
    else:
        _check(scores_out is None, "scores_out needs scores")
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
               and out.device == q.device, "invalid output tensor")
    lib, dt = _lib.load(), _DTYPES[q.dtype]
    with _DeviceGuard(q.device):
        stream = _stream_ptr(q.device)
        need = _prefix_workspace(q.device.index, B, T, H, KVH, D, prefix_length, max_length, dt,
                                 scores is not None)
        ws = workspace(q.device, stream, need, "shared_prefix")
        rc = lib.pdb_shared_prefix_attention_impl(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), prefix_table.data_ptr(),
            prefix_table.size(0), prefix_length, tables.data_ptr(), lengths.data_ptr(),
            counts.data_ptr() if counts is not None else None,
            scores.data_ptr() if width else None, scores_out.data_ptr() if width else None, width,
            out.data_ptr(), B, T, H, D, N, bs, KVH, tables.size(1), max_length, dt,
            ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
            stream, int(impl))
    _lib.check(rc, "shared_prefix_attention")
    return out if scores is None else (out, scores_out)


def verify_drafts(draft_tokens: torch.Tensor, target_probs: torch.Tensor,
                  accept_uniforms: torch.Tensor, sample_uniforms: torch.Tensor, *,
                  draft_probs: torch.Tensor | None = None,
                  draft_lengths: torch.Tensor | None = None):
    """Accept drafted tokens against the target's probabilities, draw the next one.

    draft_tokens int64 [B, T]; target_probs [B, T + 1, V] and draft_probs
    [B, T, V] (None: the drafts were not sampled, e.g. looked up) in FP32 or
    FP16; accept_uniforms fp32 [B, T] and sample_uniforms fp32 [B] are random
    numbers in [0, 1); draft_lengths int32 [B] (None: T) says how many drafts
    are real. Draft i is accepted while u_i q_i(x_i) < p_i(x_i); the next token
    is drawn from max(p - q, 0) at the first rejected draft (without
    draft_probs: p without the draft), or from p after the last one. Returns
    (tokens int64 [B, T + 1]: accepted drafts, next token, then -1; counts
    int32 [B]: accepted + 1). The draw sums 64-bit integers (weights in units
    of 2^-40), so equal inputs give equal tokens on any GPU; a row without any
    weight gives -1.
    """
    _check(target_probs.is_cuda, "probabilities must be on CUDA")
    _check_same_device(target_probs, draft_tokens, accept_uniforms, sample_uniforms, draft_probs,
                       draft_lengths)
    _check(draft_tokens.dim() == 2 and target_probs.dim() == 3, "invalid probabilities shape")
    B, T = draft_tokens.shape
    V = target_probs.size(2)
    _check(B > 0 and T > 0 and V > 0 and target_probs.shape == (B, T + 1, V),
           "invalid probabilities shape")
    _check(target_probs.dtype in _DTYPES, "use FP32 or FP16")
    if draft_probs is not None:
        _check(draft_probs.shape == (B, T, V), "invalid probabilities shape")
        _check(draft_probs.dtype == target_probs.dtype, "dtype mismatch")
    _check(draft_tokens.dtype == torch.int64, "draft tokens must be int64")
    _check(accept_uniforms.dtype == torch.float32 and accept_uniforms.shape == (B, T)
           and sample_uniforms.dtype == torch.float32 and sample_uniforms.shape == (B,),
           "invalid random numbers")
    if draft_lengths is not None:
        _check(draft_lengths.dtype == torch.int32 and draft_lengths.shape == (B,),
               "invalid draft lengths")
    tokens = torch.empty((B, T + 1), dtype=torch.int64, device=target_probs.device)
    counts = torch.empty((B,), dtype=torch.int32, device=target_probs.device)
    with _DeviceGuard(target_probs.device):
        rc = _lib.load().pdb_verify_drafts(
            draft_tokens.data_ptr(), target_probs.data_ptr(),
            draft_probs.data_ptr() if draft_probs is not None else None,
            accept_uniforms.data_ptr(), sample_uniforms.data_ptr(),
            draft_lengths.data_ptr() if draft_lengths is not None else None, tokens.data_ptr(),
            counts.data_ptr(), B, T, V, _DTYPES[target_probs.dtype],
            _stream_ptr(target_probs.device))
    _lib.check(rc, "verify_drafts")
    return tokens, counts


def evict_tokens(k: torch.Tensor, v: torch.Tensor, scores: torch.Tensor, tables: torch.Tensor,
                 lengths: torch.Tensor, new_tables: torch.Tensor, budget: int, recent: int = 0):
    """Keep ``budget`` tokens per sequence and kv head, by accumulated weight.

    k, v [blocks, block_size, KVH, D] (one layer's pools); scores fp32
    [B, KVH, S]; tables int32 [B, W] and lengths int32 [B] as in decode. The
    last ``recent`` tokens stay and, of the others, those of highest score
    (NaN lowest, equal scores by lowest index); their K and V rows go, in
    their order, to the pages ``new_tables`` int32 [B, W2] of the same pools.
    Those pages must not be in use: reserve them, evict every layer into them,
    then release the old ones (the number of kept tokens is the same in every
    layer and head). Returns (kept int32 [B, KVH, budget]: indices, then -1;
    new_lengths int32 [B]; new_scores like scores, 0 past the kept tokens).
    """
    _check(k.is_cuda, "cache must be on CUDA")
    _check_same_device(k, v, scores, tables, lengths, new_tables)
    _check(k.dim() == 4 and k.shape == v.shape and k.numel() > 0, "invalid cache shape")
    _check(k.dtype in _DTYPES, "use FP32 or FP16")
    _check(v.dtype == k.dtype, "dtype mismatch")
    N, bs, KVH, D = k.shape
    _check(lengths.dim() == 1 and lengths.size(0) > 0, "invalid lengths")
    B = lengths.size(0)
    _check(scores.dtype == torch.float32 and scores.dim() == 3 and scores.shape[:2] == (B, KVH)
           and scores.size(2) > 0, "scores must be fp32 [batch, kv_heads, tokens]")
    _check(tables.dtype == torch.int32 and lengths.dtype == torch.int32
           and new_tables.dtype == torch.int32, "metadata must be int32")
    _check(tables.dim() == 2 and tables.size(0) == B and tables.size(1) > 0
           and new_tables.dim() == 2 and new_tables.size(0) == B and new_tables.size(1) > 0,
           "invalid block tables")
    budget, recent = int(budget), int(recent)
    _check(budget > 0, "invalid budget")
    _check(0 <= recent <= budget, "recent tokens must fit the budget")
    S = scores.size(2)
    _check(new_tables.size(1) * bs >= min(budget, S, tables.size(1) * bs),
           "new tables must hold the budget")
    kept = torch.empty((B, KVH, budget), dtype=torch.int32, device=k.device)
    new_lengths = torch.empty_like(lengths)
    new_scores = torch.empty_like(scores)
    with _DeviceGuard(k.device):
        rc = _lib.load().pdb_evict_tokens(
            k.data_ptr(), v.data_ptr(), scores.data_ptr(), S, tables.data_ptr(),
            lengths.data_ptr(), new_tables.data_ptr(), kept.data_ptr(), new_lengths.data_ptr(),
            new_scores.data_ptr(), B, D, N, bs, KVH, tables.size(1), new_tables.size(1), budget,
            recent, _DTYPES[k.dtype], _stream_ptr(k.device))
    _lib.check(rc, "evict_tokens")
    return kept, new_lengths, new_scores
