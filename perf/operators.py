"""Cases, plain forms and exact values of the serving operators: attention over a
shared prefix (several query tokens per sequence, with or without accumulated
weights), verification of drafted tokens, eviction by accumulated weight.

``run`` takes what ``prepare`` made. With ``own`` false it computes an operator
from elementary torch operations in 32 bits; with ``own`` true it makes the
calls a user of the package makes.
"""
import math

import torch

own = False

#: (query heads, kv heads, head_dim) of the package's own workloads.
HEADS = {"32/8/128": (32, 8, 128), "9/3/64": (9, 3, 64)}
TYPES = {"fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


def _package():
    import importlib
    return importlib.import_module("distributed-llm-inference_b200")


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def _attention(batch, tokens, heads, dtype, prefix, shortest, longest, block_size=16, ragged=False,
               scored=False, **name):
    return dict(name, op="attention", batch=batch, tokens=tokens, heads=heads, dtype=dtype, prefix=prefix,
                shortest=shortest, longest=longest, block_size=block_size, ragged=ragged, scored=scored)


def _verify(batch, drafts, vocab, dtype, agree, given=True, **name):
    return dict(name, op="verify", batch=batch, drafts=drafts, vocab=vocab, dtype=dtype, agree=agree, given=given)


def _evict(batch, heads, dtype, shortest, longest, budget, recent, block_size=16, **name):
    return dict(name, op="evict", batch=batch, heads=heads, dtype=dtype, shortest=shortest, longest=longest,
                budget=budget, recent=recent, block_size=block_size)


def listed():
    return [
        # one user, a short instruction prefix, the first answer tokens: latency
        _attention(1, 1, "9/3/64", "fp16", 333, 1, 40, name="attention one short"),
        # a chat batch under one long instruction prefix, one token per step
        _attention(64, 1, "32/8/128", "fp16", 4096, 16, 1024, name="attention chat batch"),
        # drafted tokens scored in one pass, ragged counts, a prefix that ends inside a page
        _attention(24, 6, "32/8/128", "fp16", 2501, 8, 700, ragged=True, name="attention drafted"),
        # the small model's heads with drafts of five, larger pages
        _attention(128, 5, "9/3/64", "fp16", 1999, 5, 777, block_size=32, ragged=True, name="attention small heads"),
        # the package's 32-bit path
        _attention(16, 2, "9/3/64", "fp32", 1500, 2, 512, name="attention fp32"),
        # caches kept under a budget: weights accumulated over long own contexts, no prefix
        _attention(16, 1, "32/8/128", "fp16", 0, 2048, 8192, scored=True, name="attention accumulating"),
        # a full server: long prefix, four tokens each, long own contexts
        _attention(256, 4, "32/8/128", "fp16", 8192, 16, 2048, name="attention full server"),
        # one sequence's drafts over the vocabulary of the small model: latency
        _verify(1, 3, 49152, "fp32", 0.6, name="verify one"),
        # a batch with a weak draft model; odd vocabulary, so rows start at any alignment
        _verify(256, 5, 100003, "fp32", 0.5, name="verify batch"),
        # drafts looked up in the prompt (no draft probabilities), 16-bit probabilities
        _verify(64, 7, 49152, "fp16", 0.7, given=False, name="verify looked up"),
        # one cache just over its budget
        _evict(1, "9/3/64", "fp16", 300, 300, 256, 32, name="evict one"),
        # a server trims its caches of long own contexts
        _evict(48, "32/8/128", "fp16", 700, 8192, 1024, 128, name="evict batch"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1e15


def draw(rng):
    op = rng.choice(("attention", "attention", "verify", "evict"))
    top = max(_cost(c) for c in listed())
    if op == "attention":
        while True:
            longest = _log(rng, 1, 8192)
            case = _attention(_log(rng, 1, 256), rng.choice((1, 1, 2, 3, 4, 5, 6, 7, 8)),
                              rng.choice(sorted(HEADS)), rng.choice(("fp16", "fp16", "fp32")),
                              rng.choice((0, 1, 1, 1)) * _log(rng, 1, 8192), rng.randint(1, longest), longest,
                              rng.choice((16, 16, 32, 64)), rng.random() < 0.4, rng.random() < 0.25)
            H, KVH, D = HEADS[case["heads"]]
            B, T = case["batch"], case["tokens"]
            # the plain form's own tensors have to fit three times over too
            plain = 4.0 * B * (2 * longest * KVH * D + 2 * T * H * (longest + case["prefix"]))
            if _cost(case) <= (0.2 * top if case["dtype"] == "fp32" else top) and plain < 9e9:
                return case
    if op == "verify":
        while True:
            case = _verify(_log(rng, 1, 256), rng.randint(1, 8), _log(rng, 512, 131072), rng.choice(("fp32", "fp16")),
                           round(rng.uniform(0.2, 0.95), 2), rng.random() < 0.7)
            if case["batch"] * case["vocab"] * (case["drafts"] + 1) < 2.0e8:
                return case
    while True:
        longest = _log(rng, 32, 8192)
        budget = rng.randint(max(1, longest // 8), longest)
        case = _evict(_log(rng, 1, 96), rng.choice(sorted(HEADS)), rng.choice(("fp16", "fp16", "fp32")),
                      rng.randint(1, longest), longest, budget, rng.randint(0, budget), rng.choice((16, 16, 32, 64)))
        if _cost(case) <= top:
            return case


def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    B = case["batch"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "verify":
        rejected = 1.0 - case["agree"] ** case["drafts"]  # share of rows that read a draft row too
        rows = B * (1.0 + (rejected if case["given"] else 0.0))
        return {"bytes": rows * case["vocab"] * e + B * (case["drafts"] * (8 + 4 + 2 * e) + 8 * (case["drafts"] + 1)),
                "flops": 2.0 * B * case["vocab"]}
    H, KVH, D = HEADS[case["heads"]]
    mean = (case["shortest"] + case["longest"]) / 2
    if case["op"] == "evict":
        span = case["longest"] - case["shortest"] + 1  # lengths are uniform: the mean of min(length, budget)
        below = min(max(case["budget"] - case["shortest"], 0), span)
        kept = (below * (case["shortest"] + case["shortest"] + below - 1) / 2 + (span - below) * case["budget"]) / span
        return {"bytes": B * KVH * (4 * kept * D * e + 4 * mean + 4 * case["longest"] + 4 * case["budget"]),
                "flops": float(B * KVH * mean)}
    T = case["tokens"]
    tokens = (1 + T) / 2 if case["ragged"] else T
    mean = max(mean, tokens)
    scores = 3 * B * KVH * case["longest"] * 4 if case["scored"] else 0
    return {"bytes": 2 * B * T * H * D * e + 2 * (case["prefix"] + B * mean) * KVH * D * e + scores,
            "flops": 4.0 * tokens * H * D * B * (case["prefix"] + mean - (tokens - 1) / 2)}


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _pages(lengths, block_size, blocks, gen):
    """Tables [B, width] over a pool's randomly ordered pages, 0 beyond a sequence's own,
    and the pages that are left."""
    width = max(1, max(-(-n // block_size) for n in lengths))
    need = [-(-n // block_size) for n in lengths]
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    tables = torch.zeros(len(lengths), width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, order[at:]


def _lengths(case, gen):
    return torch.randint(case["shortest"], case["longest"] + 1, (case["batch"],), generator=gen)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    B = case["batch"]
    if case["op"] == "verify":
        return _prepare_verify(case, gen, dev, dtype)
    H, KVH, D = HEADS[case["heads"]]
    bs = case["block_size"]
    lengths = _lengths(case, gen)
    if case["op"] == "attention":
        T = case["tokens"]
        counts = torch.randint(1, T + 1, (B,), generator=gen) if case["ragged"] else torch.full((B,), T)
        lengths = torch.maximum(lengths, counts)
        prefix_pages = -(-case["prefix"] // bs)
        blocks = sum(-(-n // bs) for n in lengths.tolist()) + prefix_pages + 8
        tables, rest = _pages(lengths.tolist(), bs, blocks, gen)
        state = {"case": case, "prefix_table": rest[:prefix_pages].to(DEVICE), "prefix": case["prefix"],
                 "counts": counts.to(torch.int32).to(DEVICE) if case["ragged"] else None,
                 # heads differ in how sharply they attend
                 "q": (torch.randn(B, T, H, D, generator=dev, device=DEVICE)
                       * torch.rand(H, 1, generator=dev, device=DEVICE).mul(2.5).add(0.5)).to(dtype)}
        if case["scored"]:
            weight = torch.randn(B, KVH, case["longest"], generator=dev, device=DEVICE).mul(1.5).exp()
            state["scores"] = weight
            state["scores_out"] = torch.empty_like(weight)
    else:
        new_pages = [-(-min(n, case["budget"]) // bs) for n in lengths.tolist()]
        # room for every sequence at its longest, before and after
        blocks = B * (-(-case["longest"] // bs) + -(-min(case["longest"], case["budget"]) // bs))
        tables, rest = _pages(lengths.tolist(), bs, blocks, gen)
        width = max(1, max(new_pages))
        new_tables = torch.zeros(B, width, dtype=torch.int32)
        at = 0
        for b, n in enumerate(new_pages):
            new_tables[b, :n] = rest[at:at + n]
            at += n
        weight = torch.randn(B, KVH, case["longest"], generator=dev, device=DEVICE).mul(1.5).exp()
        # tokens that were never attended to have no weight: many equal scores
        weight *= torch.rand(B, KVH, case["longest"], generator=dev, device=DEVICE) < 0.9
        state = {"case": case, "scores": weight, "new_tables": new_tables.to(DEVICE)}
    state["k"] = torch.randn(blocks, bs, KVH, D, generator=dev, device=DEVICE, dtype=dtype)
    state["v"] = torch.randn(blocks, bs, KVH, D, generator=dev, device=DEVICE, dtype=dtype)
    state["tables"] = tables.to(DEVICE)
    state["lengths"] = lengths.to(torch.int32).to(DEVICE)
    state["max_length"] = int(lengths.max())
    return state


def _prepare_verify(case, gen, dev, dtype):
    B, T, V = case["batch"], case["drafts"], case["vocab"]

    def rows(n):  # a few likely tokens and a long tail, as a language model's output
        return torch.softmax(torch.randn(B, n, V, generator=dev, device=DEVICE).mul_(3.0), -1)

    target = rows(T + 1)
    if case["given"]:
        draft = rows(T).mul_(1 - case["agree"]).add_(target[:, :T], alpha=case["agree"])
        pick = draft
    else:
        draft, pick = None, target[:, :T]
    tokens = torch.multinomial(pick.reshape(B * T, V), 1, generator=dev).view(B, T)
    return {"case": case, "draft_tokens": tokens, "target": target.to(dtype),
            "draft": None if draft is None else draft.to(dtype),
            "accept": torch.rand(B, T, generator=dev, device=DEVICE),
            "sample": torch.rand(B, generator=dev, device=DEVICE),
            "draft_lengths": torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32).to(DEVICE)
            if B > 1 else torch.full((B,), T, dtype=torch.int32, device=DEVICE)}


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "verify": _own_verify, "evict": _own_evict}[op](state)
    return {"attention": _plain_attention, "verify": _plain_verify, "evict": _plain_evict}[op](state)


def _own_attention(s):
    return _package().shared_prefix_attention(
        s["q"], s["k"], s["v"], s["prefix_table"], s["prefix"], s["tables"], s["lengths"], s["max_length"],
        counts=s["counts"], scores=s.get("scores"), scores_out=s.get("scores_out"))


def _own_verify(s):
    return _package().verify_drafts(s["draft_tokens"], s["target"], s["accept"], s["sample"],
                                    draft_probs=s["draft"], draft_lengths=s["draft_lengths"])


def _own_evict(s):
    kept, lengths, scores = _package().evict_tokens(
        s["k"], s["v"], s["scores"], s["tables"], s["lengths"], s["new_tables"], s["case"]["budget"],
        s["case"]["recent"])
    return kept, lengths, scores, s["k"], s["v"]


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    B, T, H, D = q.shape
    bs, KVH = k.shape[1], k.shape[2]
    G = H // KVH
    dev = q.device
    P, S = s["prefix"], s["max_length"]
    pos = torch.arange(S, device=dev)
    lengths = s["lengths"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full((B,), T, device=dev)
    page = s["tables"].long()[:, pos // bs]
    live = pos < lengths[:, None]                                             # [B, S]
    own_k = torch.where(live[..., None, None], k[page, pos % bs], 0).float()  # [B, S, KVH, D]
    own_v = torch.where(live[..., None, None], v[page, pos % bs], 0).float()
    at = torch.arange(P, device=dev)
    pre_k = k[s["prefix_table"].long()[at // bs], at % bs].float()            # [P, KVH, D]
    pre_v = v[s["prefix_table"].long()[at // bs], at % bs].float()
    t = torch.arange(T, device=dev)
    real = t < counts[:, None]                                                # [B, T]
    last = lengths[:, None] - counts[:, None] + t                             # last own token that row sees
    see = real[..., None] & (pos <= last[..., None])                          # [B, T, S]
    # [KVH, B, T*G, D]: query heads of one kv head together
    x = q.float().view(B, T, KVH, G, D).permute(2, 0, 1, 3, 4).reshape(KVH, B, T * G, D)
    x = x * (1.0 / math.sqrt(D))
    logits_pre = torch.matmul(x.reshape(KVH, B * T * G, D), pre_k.permute(1, 2, 0)).view(KVH, B, T * G, P)
    logits_own = torch.matmul(x, own_k.permute(2, 0, 3, 1))                   # [KVH, B, T*G, S]
    see = see[:, :, None, :].expand(B, T, G, S).reshape(B, T * G, S)
    real = real[:, :, None].expand(B, T, G).reshape(B, T * G, 1)
    logits_own = torch.where(see, logits_own, float("-inf"))
    top = logits_own.amax(-1, keepdim=True)
    if P:
        top = torch.maximum(top, logits_pre.amax(-1, keepdim=True))
    top = torch.where(torch.isfinite(top), top, 0.0)
    w_pre = torch.where(real, torch.exp(logits_pre - top), 0.0)
    w_own = torch.exp(logits_own - top)
    total = w_pre.sum(-1, keepdim=True) + w_own.sum(-1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    out = torch.matmul(w_pre.view(KVH, B * T * G, P), pre_v.permute(1, 0, 2)).view(KVH, B, T * G, D)
    out = (out + torch.matmul(w_own, own_v.permute(2, 0, 1, 3))) / total
    out = out.view(KVH, B, T, G, D).permute(1, 2, 0, 3, 4).reshape(B, T, H, D).to(q.dtype)
    if "scores" not in s:
        return out
    added = (w_own / total).sum(2).transpose(0, 1)                            # [B, KVH, S]
    scores = s["scores"].clone()
    scores[:, :, :S] += added
    return out, scores


def _plain_verify(s):
    x, target, draft = s["draft_tokens"], s["target"], s["draft"]
    B, T = x.shape
    V = target.shape[2]
    dev = x.device
    n = s["draft_lengths"].long()
    p_x = target[:, :T].gather(2, x[..., None])[..., 0].float()
    q_x = draft.gather(2, x[..., None])[..., 0].float() if draft is not None else torch.ones_like(p_x)
    ok = (s["accept"] * q_x < p_x) & (torch.arange(T, device=dev) < n[:, None])
    accepted = torch.cumprod(ok.long(), 1).sum(1)                             # [B]
    rows = torch.arange(B, device=dev)
    rejected = accepted < n
    at = torch.clamp(accepted, max=T - 1)
    p = target[rows, accepted].float()                                        # [B, V]
    if draft is not None:
        less = torch.where(rejected[:, None], draft[rows, at].float(), 0.0)
        w = p - less
    else:
        hit = torch.arange(V, device=dev) == x[rows, at][:, None]
        w = torch.where(hit & rejected[:, None], 0.0, p)

    def fixed(a):  # parts of 2^-40: integer sums do not depend on their order
        return (torch.where(a > 0, torch.clamp(a, max=1.0), 0.0) * 2.0 ** 40).to(torch.int64)

    weight = fixed(w)
    weight = torch.where((weight.sum(1) > 0)[:, None], weight, fixed(p))
    running = torch.cumsum(weight, 1)
    total = running[:, -1]
    level = (total.double() * s["sample"].double()).to(torch.int64)
    level = torch.clamp(torch.minimum(level, total - 1), min=0)
    token = (running <= level[:, None]).sum(1)                                # first index above the level
    token = torch.where(total > 0, token, -1)
    step = torch.arange(T + 1, device=dev)
    padded = torch.cat([x, x[:, :1]], 1)
    out = torch.where(step < accepted[:, None], padded, -1)
    out = torch.where(step == accepted[:, None], token[:, None], out)
    return out, (accepted + 1).to(torch.int32)


def _plain_evict(s):
    case = s["case"]
    k, v, scores = s["k"], s["v"], s["scores"]
    B, KVH, S = scores.shape
    bs, budget = k.shape[1], case["budget"]
    dev = k.device
    lengths = s["lengths"].long()
    pos = torch.arange(S, device=dev)
    live = pos < lengths[:, None]
    recent = live & (pos >= (lengths - case["recent"])[:, None])
    rank = torch.where(torch.isnan(scores), float("-inf"), scores)
    # recent tokens first, then the others by weight (ties: lowest index), then what is no token
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    group = torch.where(recent, 0, torch.where(live, 1, 2))[:, None].expand(B, KVH, S)
    order = order.gather(2, torch.sort(group.gather(2, order), dim=-1, stable=True).indices)
    new_lengths = torch.clamp(lengths, max=budget)
    cap = min(budget, S)
    slot = torch.arange(cap, device=dev)
    inside = slot < new_lengths[:, None]                                      # [B, cap]
    kept = torch.where(inside[:, None], order[:, :, :cap], S).sort(-1).values  # by index; S: none
    b, c, i = torch.nonzero(inside[:, None].expand(B, KVH, cap), as_tuple=True)
    j = kept[b, c, i]
    old = s["tables"].long()[b, j // bs]
    new = s["new_tables"].long()[b, i // bs]
    k[new, i % bs, c] = k[old, j % bs, c]
    v[new, i % bs, c] = v[old, j % bs, c]
    new_scores = torch.zeros_like(scores)
    new_scores[b, c, i] = scores[b, c, j]
    index = torch.full((B, KVH, budget), -1, dtype=torch.int32, device=dev)
    index[b, c, i] = j.to(torch.int32)
    return index, new_lengths.to(torch.int32), new_scores, k, v


# --------------------------------------------------------------------------
# Exact values, in 64 bits and sequence by sequence
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "evict":
        return _exact_evict(s)
    return None  # tokens and counts: whole numbers


def _cells(pool, pages, n):
    """The first n token rows of a page list, [n, KVH, D] in 64 bits."""
    used = pages[: -(-n // pool.shape[1])].long() if n else pages[:0].long()
    return pool[used].flatten(0, 1)[:n].double()


def _exact_attention(s):
    q, k = s["q"], s["k"]
    B, T, H, D = q.shape
    KVH = k.shape[2]
    G = H // KVH
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=q.device)
    scores = s["scores"].double() if "scores" in s else None
    P = s["prefix"]
    counts = s["counts"].tolist() if s["counts"] is not None else [T] * B
    pre_k, pre_v = _cells(k, s["prefix_table"], P), _cells(s["v"], s["prefix_table"], P)
    for b, n in enumerate(s["lengths"].tolist()):
        c = counts[b]
        keys = torch.cat([pre_k, _cells(k, s["tables"][b], n)])
        vals = torch.cat([pre_v, _cells(s["v"], s["tables"][b], n)])
        place = torch.arange(P + n, device=q.device)
        limit = P + n - c + torch.arange(c, device=q.device)
        x = q[b, :c].double().view(c, KVH, G, D)
        a = torch.einsum("tcgd,jcd->tcgj", x, keys) / D ** 0.5
        a = a.masked_fill((place > limit[:, None])[:, None, None], float("-inf"))
        p = torch.softmax(a, -1)
        out[b, :c] = torch.einsum("tcgj,jcd->tcgd", p, vals).reshape(c, H, D)
        if scores is not None:
            scores[b, :, :n] += p[..., P:].sum((0, 2))
    return out if scores is None else (out, scores)


def _exact_evict(s):
    case = s["case"]
    scores = s["scores"].double()
    B, KVH, S = scores.shape
    k, v = s["k"].double(), s["v"].double()
    bs = k.shape[1]
    new_scores = torch.zeros_like(scores)
    for b, n in enumerate(s["lengths"].tolist()):
        m = min(n, case["budget"])
        r = min(case["recent"], m)
        where = torch.arange(m, device=k.device)
        to = s["new_tables"][b].long()[where // bs]
        for c in range(KVH):
            best = torch.sort(-scores[b, c, :n - r], stable=True).indices[: m - r]
            keep = torch.cat([best.sort().values, torch.arange(n - r, n, device=k.device)])
            frm = s["tables"][b].long()[keep // bs]
            k[to, where % bs, c] = k[frm, keep % bs, c]
            v[to, where % bs, c] = v[frm, keep % bs, c]
            new_scores[b, c, :m] = scores[b, c, keep]
    return None, None, new_scores, k, v
