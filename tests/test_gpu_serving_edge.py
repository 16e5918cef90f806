"""The serving operators where their kernels could lose bits, marks or order:
weights between two FP16 numbers, values that are not finite, calls from several
threads, launches past a grid's limits, paths that only large calls take.

Each bound is derived at its test; inputs and calls as in test_gpu_serving_ops.
"""
from __future__ import annotations

import threading
import time

import pytest
import torch

import serving_oracle as oracle
from conftest import import_module
from test_gpu_serving_ops import IMPLS, TOL, call, drafts, impl_of, make, verify

pytestmark = pytest.mark.gpu


# ---- calls from several threads ------------------------------------------------
def in_threads(jobs):
    """Runs the callables at the same time; raises what any of them raised."""
    errors = []

    def guarded(job):
        try:
            job()
        except BaseException as e:  # noqa: BLE001 - handed to the caller
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


@pytest.mark.parametrize("op", ["mma", "tcgen05", "decode", "prefill"])
def test_first_call_of_a_thread(pkg, cuda, op):
    # a new thread has no CUDA context bound: encoding tensor maps needs one
    d = make(3, 2, 8, 2, 64, torch.float16, 30, [4, 20, 67], stale=0.0)
    c = {n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()}
    one, out = c["q"][:, 0].contiguous(), torch.empty_like(c["q"])
    first = torch.empty_like(one)

    def job():
        if op == "decode":
            pkg.paged_attention(one, c["k"], c["v"], c["tables"], c["lengths"], 67, out=first)
        elif op == "prefill":
            pkg.prefill_attention(c["q"], c["k"], c["v"], c["tables"],
                                  c["lengths"].clamp(max=2), out=out)
        else:
            pkg.shared_prefix_attention(c["q"], c["k"], c["v"], c["prefix_table"], 30, c["tables"],
                                        c["lengths"], 67, out=out, impl=impl_of(pkg, op))
    job()
    torch.cuda.synchronize()
    want = [first.clone(), out.clone()]
    first.zero_(), out.zero_()
    in_threads([job])
    torch.cuda.synchronize()
    assert torch.equal(first, want[0] if op == "decode" else torch.zeros_like(first))
    assert torch.equal(out, torch.zeros_like(out) if op == "decode" else want[1])


# ---- the weights' precision ----------------------------------------------------
@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 3, 6, 16])
def test_weights_keep_more_than_sixteen_bits(pkg, cuda, T, D, impl):
    # Half of the keys have weight 1 and value 1, half a weight w in (0.5, 0.53) and
    # a value near -1 / w: the outputs are small, so that FP16 rounds them by
    # 2^-11 of little, and an error of the weights shows. One FP16 number per weight
    # is off by up to 2^-12, 3e-4 of an output. Allowed beside the output's rounding:
    # two FP16 terms 2^-21, the exponential 2^-22 and the logit 2^-23 of a weight
    # (1e-6, times values of 2), sums of 500 terms in FP32 1.5e-6.
    B, G, KVH, prefix = 12, 4, 2, 200
    lengths = [T + 21 * b for b in range(B)]
    d = make(B, T, G * KVH, KVH, D, torch.float16, prefix, lengths)
    g = torch.Generator().manual_seed(9)
    d["q"].zero_()
    d["q"][..., 0] = (torch.rand(B, T, G * KVH, generator=g) * 0.05 + 0.64) * D ** 0.5 / 2  # ln 2 = 0.693
    used = [(d["prefix_table"], prefix)] + [(d["tables"][b], n) for b, n in enumerate(lengths)]
    for table, n in used:
        for t in range(n):
            at = int(table[t // 16]), t % 16
            d["k"][at], d["v"][at] = 0.0, 1.0
            if t % 2:
                d["k"][at][:, 0] = -2.0
                d["v"][at] = -(torch.rand(KVH, D, generator=g) * 0.1 + 1.88).half()
    got = call(pkg, d, cuda, impl).cpu().double()
    want, _ = oracle.shared_prefix_attention(d["q"], d["k"], d["v"], d["prefix_table"], prefix,
                                             d["tables"], d["lengths"])
    over = (got - want).abs() - want.abs() * 2.0 ** -11
    assert over.max().item() <= 4e-6


# ---- values that are not finite ------------------------------------------------
def poison(d, b, token, dim, value, what="v"):
    """One dim of own token `token` of sequence b, every kv head."""
    d[what][int(d["tables"][b, token // 16]), token % 16, :, dim] = value


@pytest.mark.parametrize("dtype, impl", [(torch.float32, "auto"), (torch.float32, "simt")]
                         + [(torch.float16, i) for i in IMPLS])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [2, 4, 7, 10, 20])
def test_a_drafted_value_that_is_not_finite(pkg, cuda, T, D, dtype, impl):
    # V alone (the logits stay finite): the rows that see the token get it, the others
    # keep their bits. Drafted tokens in the first tile of a key range, in the
    # first, and in a later range; 4 T rows per kv head.
    lengths = [T, T + 3, T + 30, T + 140, T + 411]
    d = make(len(lengths), T, 8, 2, D, dtype, 30, lengths)
    clean = call(pkg, d, cuda, impl).cpu()
    for first in (T - 1, T // 2):  # the rows from this one on see the token
        e = dict(d, v=d["v"].clone())
        for b, n in enumerate(lengths):
            poison(e, b, n - T + first, 3, float("inf"))
            poison(e, b, n - T + first, 5, float("nan"))
        for _ in range(5):
            got = call(pkg, e, cuda, impl).cpu()
            assert torch.equal(got[:, :first], clean[:, :first])
            assert (got[:, first:, :, 3] == float("inf")).all()
            assert got[:, first:, :, 5].isnan().all()
            keep = [i for i in range(D) if i not in (3, 5)]
            # the same sums in another order and arithmetic: twice the bound of one result
            top = d["v"][d["v"] == d["v"]].abs().max().item()
            assert (got[..., keep] - clean[..., keep]).abs().max().item() <= 2 * TOL[dtype] * top
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,H,KVH,B", [(1, 4, 2, 2), (3, 8, 1, 2), (7, 16, 1, 2), (2, 8, 2, 40), (1, 9, 3, 5)])
def test_infinities_that_every_row_sees_fp16(pkg, cuda, T, H, KVH, B, D, impl):
    # as in FP32 arithmetic: an infinite v goes into its own dim only, whether its weight is
    # a few bits long, or far below FP16's range; a key whose logit is -inf has no weight
    lengths = [T + 37 + b % 3 for b in range(B)]
    d = make(B, T, H, KVH, D, torch.float16, 150, lengths)
    d["q"][..., 1], d["q"][..., 2] = d["q"][..., 1].abs() + 0.5, 1.0
    for where, table, keys in [("prefix", d["prefix_table"], (5, 40, 140))] + [
            ("own", t, (0, 3, 34)) for t in d["tables"]]:
        at = [(int(table[n // 16]), n % 16) for n in keys]
        d["v"][at[0]][:, 3 if where == "prefix" else 7] = float("inf" if where == "prefix" else "-inf")
        d["k"][at[1]][:, 1] = float("-inf")
        d["v"][at[2]][:, 9 if where == "prefix" else 11] = float("inf")
        d["k"][at[2]][:, 2] = -240.0  # a weight of 2^-30 (D 128) or 2^-43, of those near 1
    d["v"][int(d["prefix_table"][0]), 7, :, 13] = float("nan")
    out = call(pkg, d, cuda, impl).cpu()
    ref, _ = oracle.shared_prefix_attention(d["q"], d["k"], d["v"], d["prefix_table"], 150,
                                            d["tables"], d["lengths"])
    for dim, value in ((3, "inf"), (7, "-inf"), (9, "inf"), (11, "inf")):
        assert (out[..., dim] == float(value)).all(), dim
    assert out[..., 13].isnan().all()
    keep = [i for i in range(D) if i not in (3, 7, 9, 11, 13)]
    top = d["v"][torch.isfinite(d["v"])].abs().max().item()
    assert (out[..., keep].double() - ref[..., keep]).abs().max().item() <= TOL[out.dtype] * top
    assert pkg.read_device_errors() == 0


# ---- scratch that calls share ------------------------------------------------------
def test_a_call_is_issued_whole(pkg, cuda, monkeypatch):
    # a library that launches nothing and says when two calls of one stream overlap
    lib, state = import_module("_lib"), dict(inside=0, overlapped=False, calls=0)
    real = lib.load()

    class Quiet:
        def __getattr__(self, name):
            return getattr(real, name)

        def issue(self, *args):
            state["inside"] += 1
            state["overlapped"] |= state["inside"] > 1
            time.sleep(0.02)
            state["inside"] -= 1
            state["calls"] += 1
            return 0
        pdb_shared_prefix_attention_impl = pdb_rope_kv_write = pdb_paged_attention_impl = issue

    d = make(3, 2, 8, 2, 64, torch.float16, 30, [4, 20, 67])
    quiet = Quiet()
    monkeypatch.setattr(lib, "load", lambda: quiet)
    q = torch.zeros(3, 8, 64, dtype=torch.float16, device=cuda)
    pool = torch.zeros(8, 16, 2, 64, dtype=torch.float16, device=cuda)
    ints = torch.zeros(3, 4, dtype=torch.int32, device=cuda)
    long = torch.zeros(3, dtype=torch.long, device=cuda)
    inv_freq, kv = torch.ones(32, device=cuda), torch.zeros_like(q[:, :2].contiguous())
    for job in (lambda: call(pkg, d, cuda),
                lambda: pkg.paged_attention(q, pool, pool, ints, ints[:, 0].contiguous(), 64),
                lambda: pkg.rope_kv_write(q, kv, kv, pool, pool, long, long, long[:, None], inv_freq)):
        state.update(inside=0, overlapped=False, calls=0)
        in_threads([job] * 4)
        assert state["calls"] == 4 and not state["overlapped"]


def test_threads_that_share_a_stream(pkg, cuda):
    jobs = [make(20, 3, 8, 2, 64, dtype, 300, [5 + 3 * i for i in range(20)], seed=s, scores=True)
            for s, dtype in enumerate([torch.float16, torch.float16, torch.float32])]
    alone = [call(pkg, d, cuda) for d in jobs]
    inputs = [{n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()} for d in jobs]
    torch.cuda.synchronize()
    got = [[] for _ in jobs]

    def repeat(c, results):
        for _ in range(60):
            results.append(pkg.shared_prefix_attention(
                c["q"], c["k"], c["v"], c["prefix_table"], c["prefix"], c["tables"], c["lengths"],
                c["max_length"], scores=c["scores"], scores_out=torch.empty_like(c["scores"])))
    in_threads([lambda c=c, r=r: repeat(c, r) for c, r in zip(inputs, got)])
    torch.cuda.synchronize()
    for want, results in zip(alone, got):
        assert len(results) == 60
        assert all(torch.equal(x, want[0]) and torch.equal(y, want[1]) for x, y in results)


# ---- sizes past a limit of the launch -------------------------------------------
def test_accumulated_weights_of_very_many_heads(pkg, cuda):
    # batch x kv heads above 65535; the sequences share a few pages, which are read only
    B, H, KVH, D, width = 8200, 16, 8, 64, 24
    g = torch.Generator().manual_seed(4)
    d = make(1, 1, H, KVH, D, torch.float16, 20, [16 * 40])
    d.update(q=torch.randn(B, 1, H, D, generator=g).half(), max_length=width,
             tables=d["tables"][0][torch.randint(0, 40, (B, 2), generator=g)],
             lengths=torch.randint(0, width + 1, (B,), generator=g).to(torch.int32),
             scores=torch.rand(B, KVH, width + 5, generator=g))
    out, scores = call(pkg, d, cuda)
    some = [0, 1, 4095, 4096, 8190, 8191, 8192, 8199]
    want, want_scores = oracle.shared_prefix_attention(
        d["q"][some], d["k"], d["v"], d["prefix_table"], 20, d["tables"][some], d["lengths"][some],
        None, d["scores"][some])
    top = d["v"][d["v"] == d["v"]].abs().max().item()
    assert (out.cpu()[some].double() - want).abs().max().item() <= TOL[torch.float16] * top
    torch.testing.assert_close(scores.cpu()[some].double(), want_scores, rtol=2e-5, atol=2e-6)
    for part in (slice(0, 4100), slice(4100, B)):  # the same in two calls
        _, half = call(pkg, dict(d, **{n: d[n][part] for n in ("q", "tables", "lengths", "scores")}), cuda)
        torch.testing.assert_close(scores[part], half, rtol=4e-5, atol=4e-6)
    assert pkg.read_device_errors() == 0


# ---- paths that only large calls take ------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, T, own", [(621, 1, 0), (297, 4, 9)])
def test_tcgen05_ranges_that_cross_items(pkg, cuda, B, T, own, D):
    # 80 and 152 pairs of query tiles, 4 key tiles each, cut into one range per CTA: most
    # CTAs work on the end of one pair and the start of the next. The last pair is not full, the
    # prefix ends inside a tile.
    lengths = [T + b % (own - T + 1) if own else 0 for b in range(B)]
    d = make(B, T, 32, 8, D, torch.float16, 500, lengths)
    got, beside = (call(pkg, d, cuda, impl).cpu().double() for impl in ("tcgen05", "mma"))
    some = [0, 1, 15, 16, 17, B // 3, B // 2, B - 18, B - 17, B - 2, B - 1]
    want, _ = oracle.shared_prefix_attention(d["q"][some], d["k"], d["v"], d["prefix_table"], 500,
                                             d["tables"][some], d["lengths"][some])
    top = d["v"][d["v"] == d["v"]].abs().max().item()
    assert (got[some] - want).abs().max().item() <= TOL[torch.float16] * top
    assert (got - beside).abs().max().item() <= 2 * TOL[torch.float16] * top  # every row
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("B, V, dtype, given", [
    (300, 140011, torch.float16, False), (300, 140011, torch.float16, True),
    (1, 8 * 131072 + 1003, torch.float32, True), (1, 1 << 22, torch.float16, False)])
def test_verify_blocks_of_several_rounds(pkg, cuda, B, V, dtype, given):
    # more than 512 blocks of 256 entries per CTA: blocks of 512 and up to 1024 entries
    g = torch.Generator(device=cuda).manual_seed(V)
    target = torch.rand(B, 2, V, generator=g, device=cuda).pow_(4)
    target = target.div_(target.sum(-1, keepdim=True)).mul_(3000 if dtype == torch.float16 else 1).to(dtype)
    draft = target[:, :1].flip(-1).contiguous() if given else None
    tokens = torch.randint(0, V, (B, 1), generator=g, device=cuda)
    accept, sample = (torch.rand(s, generator=g, device=cuda) for s in ((B, 1), (B,)))
    sample[:3] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.999])[:B].to(cuda)
    got, counts = pkg.verify_drafts(tokens, target, accept, sample, draft_probs=draft)
    some = [b for b in (0, 1, 2, 3, 150, 299) if b < B]
    want, want_counts = oracle.verify_drafts(
        tokens[some].cpu(), target[some].cpu(), accept[some].cpu(), sample[some].cpu(),
        draft[some].cpu() if given else None)
    assert torch.equal(got.cpu()[some], want) and torch.equal(counts.cpu()[some], want_counts)
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("given", [True, False])
def test_verified_tokens_follow_the_target(pkg, cuda, given):
    # what the rule is for: whatever was drafted, the tokens are the target's. 40000 trials;
    # chi-square with 6 degrees of freedom is above 36 with probability 3e-6
    B, V = 40000, 7
    g = torch.Generator().manual_seed(8)
    p = torch.softmax(torch.randn(3, V, generator=g), -1)
    q = torch.softmax(torch.randn(2, V, generator=g), -1)
    tokens = torch.stack([torch.multinomial(q[i], B, replacement=True, generator=g) for i in range(2)], 1)
    if not given:
        tokens = torch.tensor([2, 5]).expand(B, 2).contiguous()
    out, counts = verify(pkg, dict(
        draft_tokens=tokens, target=p.expand(B, 3, V).contiguous(),
        draft=q.expand(B, 2, V).contiguous() if given else None,
        accept=torch.rand(B, 2, generator=g), sample=torch.rand(B, generator=g), draft_lengths=None), cuda)
    for place in range(3):
        there = out[counts > place, place]
        expected = p[place].double() * len(there)
        assert expected.min() > 5  # what the chi-square approximation asks for
        seen = torch.bincount(there, minlength=V).double()
        assert ((seen - expected) ** 2 / expected).sum() < 36
