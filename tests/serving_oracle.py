"""Plain 64-bit forms of the serving operators, sequence by sequence (tests only)."""
from __future__ import annotations

import math

import torch


def cells(pool, pages, n):
    """The first n token rows of a page list, [n, KVH, D] in 64 bits."""
    bs = pool.shape[1]
    rows = [pool[int(pages[t // bs]), t % bs] for t in range(n)]
    return torch.stack(rows).double() if rows else pool.new_zeros((0,) + pool.shape[2:]).double()


def shared_prefix_attention(q, k, v, prefix_table, prefix, tables, lengths, counts=None,
                            scores=None):
    """All tensors on the CPU; q [B, T, H, D]. A row's softmax runs over the keys
    that it sees and over nothing else. Returns (out fp64, scores fp64 or None)."""
    B, T, H, D = q.shape
    KVH = k.shape[2]
    G = H // KVH
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    acc = scores.double().clone() if scores is not None else None
    pk, pv = cells(k, prefix_table, prefix), cells(v, prefix_table, prefix)
    for b in range(B):
        n = int(lengths[b])
        c = int(counts[b]) if counts is not None else T
        ok, ov = cells(k, tables[b], n), cells(v, tables[b], n)
        for t in range(c):
            own = max(0, n - c + t + 1)
            kk, vv = torch.cat([pk, ok[:own]]), torch.cat([pv, ov[:own]])
            if kk.shape[0] == 0:
                continue
            for h in range(H):
                s = kk[:, h // G] @ q[b, t, h].double() / math.sqrt(D)
                p = torch.softmax(s, 0)
                out[b, t, h] = p @ vv[:, h // G]
                if acc is not None:
                    acc[b, h // G, :own] += p[prefix:]
    return out, acc


def verify_drafts(draft_tokens, target, accept, sample, draft=None, draft_lengths=None):
    """Token by token with Python integers; all tensors on the CPU."""
    B, T = draft_tokens.shape
    V = target.shape[2]
    tokens, counts = torch.full((B, T + 1), -1, dtype=torch.int64), torch.zeros(B, dtype=torch.int32)

    def fixed(w):
        return [int(min(x, 1.0) * 2 ** 40) if x > 0 else 0 for x in w.tolist()]

    for b in range(B):
        n = T if draft_lengths is None else int(draft_lengths[b])
        a = 0
        while a < n:
            x = int(draft_tokens[b, a])
            if not 0 <= x < V:
                break
            p = target[b, a, x].float()
            q = draft[b, a, x].float() if draft is not None else torch.tensor(1.0)
            if not accept[b, a] * q < p:
                break
            tokens[b, a] = x
            a += 1
        p = target[b, a].float()
        w = p.clone()
        if a < n:
            if draft is not None:
                w = p - draft[b, a].float()
            elif 0 <= int(draft_tokens[b, a]) < V:
                w[int(draft_tokens[b, a])] = 0.0
        weights = fixed(w)
        if sum(weights) == 0:
            weights = fixed(p)
        total = sum(weights)
        counts[b] = a + 1
        if total == 0:
            continue
        level = int(float(total) * float(sample[b]))
        level = max(0, min(level, total - 1))
        run = 0
        for j, x in enumerate(weights):
            run += x
            if run > level:
                tokens[b, a] = j
                break
    return tokens, counts


def evict_tokens(scores, lengths, budget, recent):
    """kept [B, KVH] lists of indices."""
    B, KVH, _ = scores.shape
    kept = []
    for b in range(B):
        n = int(lengths[b])
        m = min(n, budget)
        r = min(recent, m)
        row = []
        for c in range(KVH):
            s = [x if x == x else -math.inf for x in scores[b, c, :n - r].tolist()]
            best = sorted(range(n - r), key=lambda j: (-s[j], j))[: m - r]
            row.append(sorted(best) + list(range(n - r, n)))
        kept.append(row)
    return kept
