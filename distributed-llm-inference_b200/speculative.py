"""Speculative decoding of requests that share a prefix, on a bounded cache.

``PrefixBatch`` drives a ``PagedLlama`` through the serving operators: a prefix
that every request shares (an instruction, few-shot examples) is prefilled
once; each step scores every request's drafted tokens in one pass over the
layers (``shared_prefix_attention``: the prefix's K and V are read once for the
batch), accepts drafts against the model's probabilities (``verify_drafts``)
and, when a request's own cache passes its budget, keeps its most attended
tokens (``evict_tokens``, on the weights that the tokens which stayed gave them). The
reference decodes one token per request and step over whole contexts.

Cached keys carry RoPE at the position where their token was seen, so a cache
that lost tokens keeps the others' positions; a request's next position is
counted apart from its cache length.
"""
from __future__ import annotations

import contextlib
import itertools
import warnings

import torch

from .ops import rope_kv_write
from .serving_ops import evict_tokens, shared_prefix_attention, verify_drafts

_groups = itertools.count()  # a number of its own for each PrefixBatch: its pages' ids

# Bytes of scratch that one attention call may take, about (partial sums, and with scores
# every row's logits over the own tokens, which grow with the square of a prompt):
# longer runs of tokens are scored piece by piece. Each piece sees those before it in the cache.
_SCRATCH = 512 << 20


class PrefixBatch:
    """Requests ``ids`` that continue ``prefix`` (token ids), up to ``max_own``
    cached own tokens each. With ``budget`` a request's own cache is cut to
    that many tokens per layer and kv head whenever a step left it longer; the
    last ``recent`` stay in any case. Pages for one request's budget are kept in
    reserve for that; with more free pages more requests are cut at a time."""

    def __init__(self, runner, prefix, ids, max_own: int, budget: int | None = None,
                 recent: int = 32):
        if budget is not None and not (0 <= recent <= budget <= max_own and budget > 0):
            raise ValueError("recent <= budget <= max_own is needed")
        self.vocab = runner.model.model.embed_tokens.num_embeddings
        self._check_tokens(prefix)
        self.runner, self.ids, self.max_own = runner, list(ids), max_own
        self.budget, self.recent, self.prefix_length = budget, recent, len(prefix)
        cache, self._reserved = runner.cache, []
        prefix_id = ("shared prefix", next(_groups))

        def reserve(rid, tokens, what):
            if not cache.reserve(rid, tokens):
                raise RuntimeError(f"the cache has no pages for the {what}")
            self._reserved.append(rid)
        try:
            if prefix:
                reserve(prefix_id, len(prefix), "prefix")
                runner.prefill([prefix_id], [list(prefix)])
            self.prefix_table = torch.tensor(cache.tables.get(prefix_id, []), dtype=torch.int32,
                                             device=runner.device)
            for rid in self.ids:
                reserve(rid, max_own, "requests")
            self._spare = None  # pages that the next request is cut into
            if budget is not None and budget < max_own:
                self._spare = (*prefix_id, "spare")
                reserve(self._spare, budget, "eviction")
            layers = len(runner.model.model.layers)
            self.scores = torch.zeros((layers, len(self.ids), runner.kv_heads, max_own),
                                      device=runner.device) if budget is not None else None
        except BaseException:
            self.close()
            raise
        self.seen = {rid: 0 for rid in self.ids}  # own tokens so far, evicted ones included

    def close(self) -> None:
        """Releases the pages that this group reserved (once)."""
        for rid in self._reserved:
            self.runner.cache.release(rid)
        self._reserved = []

    def _check_tokens(self, tokens) -> None:
        # an index outside the embedding is a fault on the GPU
        if not all(0 <= t < self.vocab for t in tokens):
            raise ValueError("token outside the vocabulary")

    @contextlib.contextmanager
    def _unchanged_by_failure(self):
        """What fails inside (no memory, a refused argument) leaves the requests as they
        were. Scores are replaced, never changed in place; cells past a request's
        length may hold anything."""
        cache, seen, scores = self.runner.cache, dict(self.seen), self.scores
        lengths = {rid: cache.lengths[rid] for rid in self.ids}
        try:
            yield
        except BaseException:
            cache.lengths.update(lengths)
            self.seen, self.scores = seen, scores
            raise

    @torch.inference_mode()
    def score(self, token_lists, last_only: bool = False) -> torch.Tensor:
        """Appends each request's tokens (one or more, ragged) to its cache and
        returns the logits that follow them, float32 [B, T, vocab] (rows past a
        request's own count are meaningless). With ``last_only`` the LM head runs
        on each request's last token alone, and its logits are returned,
        [B, vocab]: for prompts, whose other logits nobody reads."""
        with self._unchanged_by_failure():
            return self._score(token_lists, last_only=last_only)

    def _piece(self, longest: int, scored: bool) -> int:
        """Tokens per request that one attention call takes."""
        runner = self.runner
        per_token = 4 * len(self.ids) * runner.heads * (2 * runner.head_dim
                                                        + (longest if scored else 0))
        return max(1, min(4096, _SCRATCH // per_token))  # 4096: the operator's own limit

    def _logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return self.runner.model.lm_head(hidden).float()

    def _score(self, token_lists, queries: list | None = None, last_only: bool = False):
        """``score``; with ``queries`` each layer's rotated queries are added to that
        list, and no weights to the scores."""
        lengths, counts = self.runner.cache.lengths, [len(tokens) for tokens in token_lists]
        if len(counts) != len(self.ids):
            raise ValueError("each request needs its tokens")
        for tokens in token_lists:
            self._check_tokens(tokens)
        after = [lengths[rid] + n for rid, n in zip(self.ids, counts)]
        if any(not n for n in counts) or max(after) > self.max_own:
            raise ValueError("each request takes one token at least, and max_own cached in all")
        T, size = max(counts), self._piece(max(after), queries is None and self.scores is not None)
        out, kept = None, []
        for t0 in range(0, T, size):
            piece, kept_here = [tokens[t0:t0 + size] for tokens in token_lists], []
            hidden = self._forward(piece, None if queries is None else kept_here)
            kept.append(kept_here)
            if last_only:  # the hidden states of the last tokens, from the pieces they are in
                ends = [b for b, n in enumerate(counts) if t0 < n <= t0 + size]
                out = hidden.new_empty((len(counts), hidden.shape[2])) if out is None else out
                out[ends] = hidden[ends, [counts[b] - 1 - t0 for b in ends]]
            elif T <= size:
                out = self._logits(hidden)
            else:
                part = self._logits(hidden)
                out = part.new_empty((part.shape[0], T, part.shape[2])) if out is None else out
                out[:, t0:t0 + size] = part
        if queries is not None:
            queries += [torch.cat(parts, 1) for parts in zip(*kept)] if len(kept) > 1 else kept[0]
        return self._logits(out) if last_only else out

    def _forward(self, token_lists, queries: list | None) -> torch.Tensor:
        """One pass over the layers, to the normed hidden states [B, T, hidden]; requests
        may have no token in it."""
        runner, cache = self.runner, self.runner.cache
        counts = [len(tokens) for tokens in token_lists]
        B, T = len(self.ids), max(counts)
        before = [cache.lengths[rid] for rid in self.ids]
        rows = torch.tensor([list(t) + [0] * (T - len(t)) for t in token_lists])
        first = torch.tensor([self.prefix_length + self.seen[rid] for rid in self.ids])
        positions = (first[:, None] + torch.arange(T)).to(runner.device)
        valid = (torch.arange(T) < torch.tensor(counts)[:, None]).to(runner.device)
        physical, offsets = cache.slots(self.ids, [range(b, b + n) for b, n in zip(before, counts)])
        for rid, b, n in zip(self.ids, before, counts):
            cache.lengths[rid] = b + n
            self.seen[rid] += n
        tables, lengths, longest = cache.metadata(self.ids)
        real = torch.tensor(counts, dtype=torch.int32, device=runner.device)
        scores = self.scores if queries is None else None
        new_scores = torch.empty_like(scores) if scores is not None else None
        x = runner.model.model.embed_tokens(rows.to(runner.device))
        for index, layer in enumerate(runner.model.model.layers):
            attn = layer.self_attn
            h = layer.input_layernorm(x)
            q = attn.q_proj(h).view(B, T, runner.heads, runner.head_dim)
            k = attn.k_proj(h).view(B, T, runner.kv_heads, runner.head_dim)
            v = attn.v_proj(h).view(B, T, runner.kv_heads, runner.head_dim)
            keys, values = cache.keys[index], cache.values[index]
            q, _ = rope_kv_write(q, k, v.contiguous(), keys, values, physical, offsets, positions,
                                 runner.inv_freq, valid=valid, inplace=True)
            context = shared_prefix_attention(
                q, keys, values, self.prefix_table, self.prefix_length, tables, lengths, longest,
                counts=real, **self._scored(scores, new_scores, index))
            if scores is not None:
                context = context[0]
            if queries is not None:
                queries.append(q)
            x = x + attn.o_proj(context.reshape(B, T, -1))
            x = x + layer.mlp(layer.post_attention_layernorm(x))
        if scores is not None:
            self.scores = new_scores
        return runner.model.model.norm(x)

    @staticmethod
    def _scored(scores, new_scores, index) -> dict:
        if scores is None:
            return {}
        return dict(scores=scores[index], scores_out=new_scores[index])

    def _accumulate(self, queries, counts) -> None:
        """Adds the weights that each request's first ``counts`` query rows give, now that
        its cache ends with those tokens. The other rows were rejected drafts, whose
        weights would rank tokens by a text that is not there."""
        cache = self.runner.cache
        tables, lengths, longest = cache.metadata(self.ids)
        real = torch.tensor(counts, dtype=torch.int32, device=self.runner.device)
        T, size = queries[0].shape[1], self._piece(longest, True)
        for t0 in range(0, T, size):
            here = (real - t0).clamp(0, size)  # a request's rows of this piece, and its
            ends = lengths - (real - t0 - here).clamp(min=0)  # length with them
            new_scores = torch.empty_like(self.scores)
            for index, q in enumerate(queries):
                shared_prefix_attention(q[:, t0:t0 + size].contiguous(), cache.keys[index],
                                        cache.values[index], self.prefix_table,
                                        self.prefix_length, tables, ends, longest, counts=here,
                                        **self._scored(self.scores, new_scores, index))
            self.scores = new_scores

    @torch.inference_mode()
    def step(self, last_tokens, drafts, accept_uniforms, sample_uniforms, draft_probs=None,
             temperature: float = 1.0):
        """One speculative step. ``last_tokens``: each request's newest token,
        not cached yet; ``drafts``: up to T guessed tokens after it;
        ``accept_uniforms`` fp32 [B, T], ``sample_uniforms`` fp32 [B];
        ``draft_probs`` fp32 [B, T, vocab], or None for drafts that were not
        sampled. Returns the new tokens of each request (1 to T + 1 of them):
        distributed as the model's own over what is cached, however good the drafts
        are. With a budget the attention runs a second time, over the tokens that
        stayed, for the weights that eviction goes by."""
        with self._unchanged_by_failure():
            new = self._step(last_tokens, drafts, accept_uniforms, sample_uniforms, draft_probs,
                             temperature)
            over = [rid for rid in self.ids
                    if self.budget is not None and self.runner.cache.lengths[rid] > self.budget]
            over = over[self._evict_some(over):]
        try:
            self.evict(over)
        except Exception as e:  # some are cut, so the step stands; the next one cuts the rest
            warnings.warn(f"requests stay over their budget for a step: {e}")
        return new

    def _step(self, last_tokens, drafts, accept_uniforms, sample_uniforms, draft_probs, temperature):
        cache, device = self.runner.cache, self.runner.device
        if not 0.0 < temperature < float("inf"):
            raise ValueError("the temperature must be positive and finite")
        if not len(last_tokens) == len(drafts) == len(self.ids):
            raise ValueError("each request needs its last token and its drafts")
        if accept_uniforms.dim() != 2 or accept_uniforms.shape[0] != len(self.ids) or any(
                len(d) > accept_uniforms.shape[1] for d in drafts):
            raise ValueError("accept_uniforms needs a row per request, a number per draft")
        T = accept_uniforms.shape[1]
        before = [cache.lengths[rid] for rid in self.ids]
        seen = dict(self.seen)
        queries = [] if self.scores is not None else None
        logits = self._score([[a, *d] for a, d in zip(last_tokens, drafts)], queries)
        probs = torch.softmax(logits / temperature, -1)
        if probs.shape[1] < T + 1:
            probs = torch.nn.functional.pad(probs, (0, 0, 0, T + 1 - probs.shape[1]))
        tokens, counts = verify_drafts(
            torch.tensor([list(d) + [0] * (T - len(d)) for d in drafts], device=device),
            probs.contiguous(), accept_uniforms, sample_uniforms, draft_probs=draft_probs,
            draft_lengths=torch.tensor([len(d) for d in drafts], dtype=torch.int32, device=device))
        new = [row[:n] for row, n in zip(tokens.tolist(), counts.tolist())]
        if any(t < 0 for got in new for t in got):
            raise RuntimeError("the model's probabilities leave no token to draw (NaN logits?)")
        for b, (rid, got) in enumerate(zip(self.ids, new)):
            # the last token and the accepted drafts stay cached; cells past them are free
            cache.lengths[rid] = before[b] + len(got)
            self.seen[rid] = seen[rid] + len(got)
        if self.budget is not None:
            self._accumulate(queries, [len(got) for got in new])
        return new

    @torch.inference_mode()
    def evict(self, ids) -> None:
        """Cuts the own caches of ``ids`` to the budget, into fresh pages, as many at a
        time as there are pages for. Where it fails, those cut so far are cut and the
        others as they were."""
        if self._spare is None and ids:
            raise ValueError("a group without a budget below max_own evicts nothing")
        ids = list(ids)
        while ids:
            ids = ids[self._evict_some(ids):]

    def _evict_some(self, ids) -> int:
        """Cuts the first of ``ids``, and those after it that there are pages for;
        returns how many. All of them or, where it fails, none."""
        cache, reserved = self.runner.cache, []
        if not ids:
            return 0
        try:
            into = {ids[0]: self._spare}
            for rid in ids[1:]:
                if not cache.reserve((rid, "kept"), self.budget):
                    break
                into[rid] = (rid, "kept")
                reserved.append((rid, "kept"))
            ids = list(into)
            rows = torch.tensor([self.ids.index(rid) for rid in ids], device=self.scores.device)
            tables, lengths, _ = cache.metadata(ids)
            new_tables = torch.tensor([cache.tables[into[rid]] for rid in ids], dtype=torch.int32,
                                      device=tables.device)
            scores = self.scores.clone()
            for index in range(scores.shape[0]):
                _, _, kept = evict_tokens(cache.keys[index], cache.values[index],
                                          scores[index][rows], tables, lengths, new_tables,
                                          self.budget, self.recent)
                scores[index][rows] = kept
        except BaseException:
            for rid in reserved:
                cache.release(rid)
            raise
        self.scores = scores
        for rid, other in into.items():
            # the new pages, then what the old ones have beyond the budget: as many as before
            new, old = cache.tables[other], cache.tables[rid]
            cache.tables[rid], cache.tables[other] = new + old[len(new):], old[:len(new)]
            cache.lengths[rid] = min(cache.lengths[rid], self.budget)
            if other != self._spare:
                cache.release(other)
        return len(ids)
