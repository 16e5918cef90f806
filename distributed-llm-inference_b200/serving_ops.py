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
from .ops import _DTYPES, _DeviceGuard, _stream_ptr, launch_lock, workspace

_INT32, _INT64, _FP32 = torch.int32, torch.int64, torch.float32
_current_device = torch.cuda.current_device


def _refuse(message: str):
    raise RuntimeError(message)


# The checks below are plain conditions, and a tensor's properties are read once: a
# call of a few microseconds on the GPU should not wait for its arguments' checks.
def _check_same_device(device: int, *tensors) -> None:
    for t in tensors:
        if t is not None:
            if t.get_device() != device:
                _refuse("all tensors must be on the same GPU")
            if not t.is_contiguous():
                _refuse("all tensors must be contiguous")


def _run_on(device: int, launch, what: str) -> None:
    """Runs `launch` with `device` current; raises on a failed call."""
    if _current_device() == device:
        rc = launch()
    else:
        with _DeviceGuard(torch.device("cuda", device)):
            rc = launch()
    if rc:
        _lib.check(rc, what)


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
    device = q.get_device()
    if device < 0:
        _refuse("query must be on CUDA")
    _check_same_device(device, q, k, v, prefix_table, tables, lengths, counts, scores, scores_out)
    q_shape, k_shape = q.shape, k.shape
    if len(k_shape) != 4 or v.shape != k_shape:
        _refuse("invalid Q/K/V shapes")
    if len(q_shape) == 4:
        B, T, H, D = q_shape
    elif len(q_shape) == 3:
        (B, H, D), T = q_shape, 1
    else:
        _refuse("invalid Q/K/V shapes")
    N, bs, KVH, Dk = k_shape
    if not (B > 0 and T > 0 and H > 0 and 0 < D <= 256):
        _refuse("invalid query shape")
    if not (N > 0 and bs > 0 and KVH > 0 and Dk == D):
        _refuse("invalid cache shape")
    if H % KVH:
        _refuse("query heads must be a multiple of KV heads")
    dtype = q.dtype
    dt = _DTYPES.get(dtype)
    if dt is None:
        _refuse("use FP32 or FP16")
    if k.dtype != dtype or v.dtype != dtype:
        _refuse("dtype mismatch")
    if not (tables.dtype == lengths.dtype == prefix_table.dtype == _INT32):
        _refuse("metadata must be int32")
    if tables.dim() != 2 or tables.shape[0] != B or prefix_table.dim() != 1:
        _refuse("invalid block tables")
    if lengths.shape != (B,):
        _refuse("invalid lengths")
    if counts is not None and (counts.dtype != _INT32 or counts.shape != (B,)):
        _refuse("invalid token counts")
    prefix_length, max_length = int(prefix_length), int(max_length)
    pages, table_width = prefix_table.shape[0], tables.shape[1]
    if not 0 <= prefix_length <= pages * bs:
        _refuse("invalid prefix length")
    if not 0 <= max_length <= table_width * bs:
        _refuse("invalid context bound")
    width, scores_ptr, scores_out_ptr = 0, None, None
    if scores is not None:
        if scores.dtype != _FP32 or scores.dim() != 3 or scores.shape[:2] != (B, KVH):
            _refuse("scores must be fp32 [batch, kv_heads, tokens]")
        width = scores.shape[2]
        if width < max_length:
            _refuse("scores must hold max_length tokens")
        if scores_out is None:
            scores_out = scores
        elif scores_out.shape != scores.shape or scores_out.dtype != _FP32:
            _refuse("invalid scores output")
        if width:
            scores_ptr, scores_out_ptr = scores.data_ptr(), scores_out.data_ptr()
    elif scores_out is not None:
        _refuse("scores_out needs scores")
    if out is None:
        out = torch.empty_like(q)
    elif not (out.shape == q_shape and out.dtype == dtype and out.is_contiguous()
              and out.get_device() == device):
        _refuse("invalid output tensor")

    def launch():
        where = q.device
        stream = _stream_ptr(where)
        need = _prefix_workspace(device, B, T, H, KVH, D, prefix_length, max_length, dt,
                                 width > 0)
        with launch_lock(device, stream, "shared_prefix"):
            ws = workspace(where, stream, need, "shared_prefix")
            return _lib.load().pdb_shared_prefix_attention_impl(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), prefix_table.data_ptr(), pages,
                prefix_length, tables.data_ptr(), lengths.data_ptr(),
                counts.data_ptr() if counts is not None else None, scores_ptr, scores_out_ptr,
                width, out.data_ptr(), B, T, H, D, N, bs, KVH, table_width, max_length, dt,
                ws.data_ptr() if ws is not None else None, need, stream, impl)

    _run_on(device, launch, "shared_prefix_attention")
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
    device = target_probs.get_device()
    if device < 0:
        _refuse("probabilities must be on CUDA")
    _check_same_device(device, target_probs, draft_tokens, accept_uniforms, sample_uniforms,
                       draft_probs, draft_lengths)
    shape = target_probs.shape
    if draft_tokens.dim() != 2 or len(shape) != 3:
        _refuse("invalid probabilities shape")
    (B, T), V = draft_tokens.shape, shape[2]
    if not (B > 0 and T > 0 and V > 0 and shape[0] == B and shape[1] == T + 1):
        _refuse("invalid probabilities shape")
    dtype = target_probs.dtype
    dt = _DTYPES.get(dtype)
    if dt is None:
        _refuse("use FP32 or FP16")
    if draft_probs is not None:
        if draft_probs.shape != (B, T, V):
            _refuse("invalid probabilities shape")
        if draft_probs.dtype != dtype:
            _refuse("dtype mismatch")
    if draft_tokens.dtype != _INT64:
        _refuse("draft tokens must be int64")
    if not (accept_uniforms.dtype == sample_uniforms.dtype == _FP32
            and accept_uniforms.shape == (B, T) and sample_uniforms.shape == (B,)):
        _refuse("invalid random numbers")
    if draft_lengths is not None and (draft_lengths.dtype != _INT32
                                      or draft_lengths.shape != (B,)):
        _refuse("invalid draft lengths")
    tokens = draft_tokens.new_empty((B, T + 1))
    counts = (torch.empty_like(draft_lengths) if draft_lengths is not None
              else draft_tokens.new_empty((B,), dtype=_INT32))

    def launch():
        return _lib.load().pdb_verify_drafts(
            draft_tokens.data_ptr(), target_probs.data_ptr(),
            draft_probs.data_ptr() if draft_probs is not None else None,
            accept_uniforms.data_ptr(), sample_uniforms.data_ptr(),
            draft_lengths.data_ptr() if draft_lengths is not None else None, tokens.data_ptr(),
            counts.data_ptr(), B, T, V, dt, _stream_ptr(target_probs.device))

    _run_on(device, launch, "verify_drafts")
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
    device = k.get_device()
    if device < 0:
        _refuse("cache must be on CUDA")
    _check_same_device(device, k, v, scores, tables, lengths, new_tables)
    k_shape = k.shape
    if len(k_shape) != 4 or v.shape != k_shape or 0 in k_shape:
        _refuse("invalid cache shape")
    dt = _DTYPES.get(k.dtype)
    if dt is None:
        _refuse("use FP32 or FP16")
    if v.dtype != k.dtype:
        _refuse("dtype mismatch")
    N, bs, KVH, D = k_shape
    if lengths.dim() != 1 or lengths.shape[0] == 0:
        _refuse("invalid lengths")
    B = lengths.shape[0]
    s_shape = scores.shape
    if not (scores.dtype == _FP32 and len(s_shape) == 3 and s_shape[0] == B
            and s_shape[1] == KVH and s_shape[2] > 0):
        _refuse("scores must be fp32 [batch, kv_heads, tokens]")
    if not (tables.dtype == lengths.dtype == new_tables.dtype == _INT32):
        _refuse("metadata must be int32")
    t_shape, n_shape = tables.shape, new_tables.shape
    if not (len(t_shape) == 2 and t_shape[0] == B and t_shape[1] > 0
            and len(n_shape) == 2 and n_shape[0] == B and n_shape[1] > 0):
        _refuse("invalid block tables")
    budget, recent, S = int(budget), int(recent), s_shape[2]
    if budget <= 0:
        _refuse("invalid budget")
    if not 0 <= recent <= budget:
        _refuse("recent tokens must fit the budget")
    if n_shape[1] * bs < min(budget, S, t_shape[1] * bs):
        _refuse("new tables must hold the budget")
    kept = lengths.new_empty((B, KVH, budget))
    new_lengths = torch.empty_like(lengths)
    new_scores = torch.empty_like(scores)

    def launch():
        return _lib.load().pdb_evict_tokens(
            k.data_ptr(), v.data_ptr(), scores.data_ptr(), S, tables.data_ptr(),
            lengths.data_ptr(), new_tables.data_ptr(), kept.data_ptr(), new_lengths.data_ptr(),
            new_scores.data_ptr(), B, D, N, bs, KVH, t_shape[1], n_shape[1], budget, recent, dt,
            _stream_ptr(k.device))

    _run_on(device, launch, "evict_tokens")
    return kept, new_lengths, new_scores
