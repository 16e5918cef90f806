"""shared_prefix_attention, verify_drafts and evict_tokens on the GPU against
64-bit plain forms (tests/serving_oracle.py), and their refusals.

Tolerances. FP16: a weight rounded to FP16 is off by at most 2^-11 of itself and
the weights of a row sum to 1, so the output moves by at most 2^-11 max|v|;
rounding the output adds 2^-11 |out|. Logits summed in FP32 are off by a few
units of 2^-20 (|logit| < 16), which moves the output by under 1e-4 max|v|:
together below 1.3e-3 max|v|. FP32: the logits' 2^-20 and the sums of weights
and products (2^-24 each, growing as the square root of their number) stay
below 2e-5 max|v|. Accumulated weights carry the logits' error alone: 2e-5
of the weight, plus the FP32 rounding of the score they are added to.
"""
from __future__ import annotations

import math

import pytest
import torch

import serving_oracle as oracle
from conftest import import_pkg

pytestmark = pytest.mark.gpu

TOL = {torch.float16: 1.3e-3, torch.float32: 2e-5}
IMPLS = ["auto", "simt", "mma", "tcgen05"]


def impl_of(pkg, name):
    return {"auto": pkg.PREFIX_AUTO, "simt": pkg.PREFIX_SIMT, "mma": pkg.PREFIX_MMA,
            "tcgen05": pkg.PREFIX_TCGEN05}[name]


def covered(impl, dtype, D, bs):
    """The tensor-core kernels take FP16, head_dim 64 and 128, whole 16-token units."""
    return impl in ("auto", "simt") or (dtype == torch.float16 and D in (64, 128) and bs % 16 == 0)


def pages(lengths, bs, spare, gen):
    need = [-(-n // bs) for n in lengths]
    blocks = sum(need) + spare
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    tables = torch.zeros(len(lengths), max(1, max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, order[at:], blocks


def make(B, T, H, KVH, D, dtype, prefix, lengths, bs=16, counts=None, scores=False, seed=0,
         stale=float("nan"), sharp=1.0):
    """Inputs on the CPU; every pool cell that no sequence and no prefix uses holds `stale`."""
    g = torch.Generator().manual_seed(seed)
    tables, rest, blocks = pages(lengths, bs, -(-prefix // bs) + 3, g)
    prefix_table = rest[: -(-prefix // bs)]
    k = torch.full((blocks, bs, KVH, D), stale).to(dtype)
    v = torch.full((blocks, bs, KVH, D), stale).to(dtype)

    def fill(table, n):
        for t in range(n):
            k[int(table[t // bs]), t % bs] = torch.randn(KVH, D, generator=g).to(dtype)
            v[int(table[t // bs]), t % bs] = torch.randn(KVH, D, generator=g).to(dtype)

    fill(prefix_table, prefix)
    for b, n in enumerate(lengths):
        fill(tables[b], n)
    d = dict(q=(torch.randn(B, T, H, D, generator=g) * sharp).to(dtype), k=k, v=v,
             prefix_table=prefix_table, prefix=prefix, tables=tables,
             lengths=torch.tensor(lengths, dtype=torch.int32), max_length=max(lengths),
             counts=None if counts is None else torch.tensor(counts, dtype=torch.int32))
    if scores:
        d["scores"] = torch.rand(B, KVH, max(lengths) + 5, generator=g) * 3
    return d


def call(pkg, d, cuda, impl="auto", **kw):
    c = {n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()}
    return pkg.shared_prefix_attention(
        c["q"], c["k"], c["v"], c["prefix_table"], c["prefix"], c["tables"], c["lengths"],
        c["max_length"], counts=c["counts"], scores=c.get("scores"), impl=impl_of(pkg, impl), **kw)


def check(pkg, d, cuda, impl="auto"):
    if not covered(impl, d["q"].dtype, d["q"].shape[-1], d["k"].shape[1]):
        with pytest.raises(RuntimeError, match="tensor-core kernels do not support"):
            call(pkg, d, cuda, impl)
        return None
    got = call(pkg, d, cuda, impl)
    out, sc = got if "scores" in d else (got, None)
    ref, ref_sc = oracle.shared_prefix_attention(
        d["q"], d["k"], d["v"], d["prefix_table"], d["prefix"], d["tables"], d["lengths"],
        d["counts"], d.get("scores"))
    top = max(1.0, d["v"][d["v"] == d["v"]].abs().max().item() if (d["v"] == d["v"]).any() else 1.0)
    err = (out.cpu().double() - ref).abs().max().item()
    assert out.dtype == d["q"].dtype
    assert err <= TOL[out.dtype] * top, f"max abs err {err:.3e}, max|v| {top:.2f}"
    if sc is not None:
        torch.testing.assert_close(sc.cpu().double(), ref_sc, rtol=2e-5, atol=2e-6)
    assert pkg.read_device_errors() == 0
    return out


ATTENTION = {
    # name: (B, T, H, KVH, D, prefix, lengths, bs, counts)
    "one token, one key": (1, 1, 3, 3, 64, 0, [1], 16, None),
    "prefix only rows": (2, 1, 4, 2, 64, 1, [0, 1], 16, None),
    "nothing to see": (2, 2, 4, 4, 64, 0, [0, 1], 16, None),
    "no own tokens at all": (2, 1, 4, 2, 128, 40, [0, 0], 16, None),
    "page and tile edges": (5, 1, 8, 2, 128, 64, [15, 16, 17, 63, 65], 16, None),
    "prefix ends inside a page": (3, 1, 9, 3, 64, 131, [5, 64, 70], 32, None),
    "drafts": (3, 5, 8, 2, 128, 77, [5, 40, 129], 16, None),
    "ragged drafts": (4, 5, 9, 3, 64, 50, [3, 40, 129, 7], 16, [3, 1, 5, 0]),
    "fewer keys than drafts": (2, 6, 4, 2, 64, 0, [2, 6], 16, None),
    "many rows": (40, 4, 8, 2, 64, 200, [(i * 7) % 33 for i in range(40)], 16, None),
    "rows past a tile": (47, 3, 8, 2, 128, 300, [3 + i % 9 for i in range(47)], 16, None),
    "group of 3, many rows": (60, 3, 9, 3, 64, 190, [3 + i % 5 for i in range(60)], 64, None),
    "one head per kv head": (6, 2, 4, 4, 128, 90, [2, 3, 17, 33, 64, 100], 16, None),
    "sixteen heads per kv head": (3, 2, 32, 2, 64, 90, [2, 33, 100], 16, None),
    "odd block size": (3, 2, 8, 2, 64, 45, [2, 33, 100], 12, None),
    "block size 1": (2, 2, 4, 2, 64, 9, [2, 21], 1, None),
    "odd head_dim": (3, 2, 6, 2, 40, 45, [2, 33, 70], 16, None),
    "head_dim 256": (2, 3, 4, 2, 256, 45, [3, 70], 16, None),
    "head_dim 1": (2, 1, 2, 1, 1, 5, [1, 20], 16, None),
    "long": (2, 1, 8, 2, 128, 2500, [1, 1700], 16, None),
    "long drafts": (2, 8, 9, 3, 64, 1, [1500, 600], 16, None),
}


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("name", list(ATTENTION))
def test_shared_prefix_attention(pkg, cuda, name, dtype, impl):
    B, T, H, KVH, D, prefix, lengths, bs, counts = ATTENTION[name]
    check(pkg, make(B, T, H, KVH, D, dtype, prefix, lengths, bs, counts), cuda, impl)


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("name", ["one token, one key", "prefix only rows", "nothing to see",
                                  "page and tile edges", "ragged drafts", "many rows",
                                  "sixteen heads per kv head", "odd block size", "long"])
def test_accumulated_weights(pkg, cuda, name, dtype, impl):
    B, T, H, KVH, D, prefix, lengths, bs, counts = ATTENTION[name]
    check(pkg, make(B, T, H, KVH, D, dtype, prefix, lengths, bs, counts, scores=True), cuda, impl)


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_sharp_and_large_logits(pkg, cuda, dtype, impl):
    if not covered(impl, dtype, 64, 16):
        pytest.skip("the tensor-core kernels take FP16")
    # |logit| up to ~200: the running maximum has to carry the exponentials. The
    # logits' rounding grows with them: 2^-24 * 200 * sqrt(64) is still 1e-4 of a weight.
    d = make(6, 2, 8, 2, 64, dtype, 150, [2, 9, 17, 80, 33, 64], sharp=30.0)
    got = call(pkg, d, cuda, impl)
    ref, _ = oracle.shared_prefix_attention(d["q"], d["k"], d["v"], d["prefix_table"], d["prefix"],
                                            d["tables"], d["lengths"])
    top = d["v"][d["v"] == d["v"]].abs().max().item()
    tol = 1.3e-3 if dtype == torch.float16 else 2e-4
    assert (got.cpu().double() - ref).abs().max().item() <= tol * top


@pytest.mark.parametrize("impl", IMPLS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_a_later_draft_never_reaches_an_earlier_one(pkg, cuda, dtype, impl):
    if not covered(impl, dtype, 64, 16):
        pytest.skip("the tensor-core kernels take FP16")
    # infinities and NaN in the cells of later drafted tokens: earlier rows do not see them
    d = make(3, 4, 8, 2, 64, dtype, 30, [4, 20, 67])
    clean = call(pkg, d, cuda, impl).cpu()
    for bad in (float("nan"), float("inf")):
        for b, n in enumerate([4, 20, 67]):
            t = n - 1
            d["v"][int(d["tables"][b, t // 16]), t % 16] = bad
            d["k"][int(d["tables"][b, t // 16]), t % 16] = bad
        got = call(pkg, d, cuda, impl).cpu()
        assert torch.equal(got[:, :3], clean[:, :3])
        assert not torch.isfinite(got[:, 3]).any()


OWN_ROWS = {
    # name: (B, T, H, KVH, D, prefix, lengths, bs, counts); T G = 9, 16, 20, 32, 48, 80
    "9 rows": (3, 3, 9, 3, 64, 33, [3, 40, 129], 16, None),
    "16 rows": (2, 4, 8, 2, 128, 0, [4, 300], 16, [4, 2]),
    "20 rows": (2, 5, 8, 2, 64, 20, [31, 33], 1, None),
    "32 rows": (3, 8, 8, 2, 128, 100, [8, 95, 260], 16, [8, 8, 1]),
    "48 rows": (2, 12, 8, 2, 128, 10, [12, 140], 12, None),
    "80 rows": (2, 20, 8, 2, 64, 70, [19, 400], 16, [19, 20]),
}


@pytest.mark.parametrize("impl", ["auto", "simt"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("name", OWN_ROWS)
def test_rows_of_a_sequence(pkg, cuda, name, dtype, impl):
    B, T, H, KVH, D, prefix, lengths, bs, counts = OWN_ROWS[name]
    check(pkg, make(B, T, H, KVH, D, dtype, prefix, lengths, bs, counts, scores=True), cuda, impl)


@pytest.mark.parametrize("impl", ["auto", "simt"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,H,KVH,B", [(1, 4, 2, 2), (2, 8, 1, 2), (3, 8, 1, 2), (7, 16, 1, 2)])
def test_infinities_that_every_row_sees(pkg, cuda, T, H, KVH, B, D, impl):
    # FP32 arithmetic keeps them: V's go into their own dim only, and a key whose logit
    # is -inf has no weight, whatever the other keys of its tile are
    lengths = [T + 37] * B
    d = make(B, T, H, KVH, D, torch.float32, 70, lengths)
    d["q"][..., 1] = d["q"][..., 1].abs() + 0.5
    for n in (5, 40):
        at = int(d["prefix_table"][n // 16]), n % 16
        d["v"][at][:, 3] = float("inf")
        at = int(d["prefix_table"][n // 16]), (n + 1) % 16
        d["k"][at][:, 1] = float("-inf")
    for b in range(B):
        at = int(d["tables"][b, 1]), 2
        d["v"][at][:, 7] = float("-inf")
        at = int(d["tables"][b, 0]), 3
        d["k"][at][:, 1] = float("-inf")
    out = call(pkg, d, cuda, impl).cpu()
    ref, _ = oracle.shared_prefix_attention(d["q"], d["k"], d["v"], d["prefix_table"], d["prefix"],
                                            d["tables"], d["lengths"], d["counts"], None)
    assert (out[..., 3] == float("inf")).all() and (out[..., 7] == float("-inf")).all()
    keep = [i for i in range(D) if i not in (3, 7)]
    top = d["v"][torch.isfinite(d["v"])].abs().max().item()
    assert (out[..., keep].double() - ref[..., keep]).abs().max().item() <= TOL[out.dtype] * top


@pytest.mark.parametrize("name", ["nothing to see", "ragged drafts", "long drafts", "many rows"])
@pytest.mark.parametrize("impl", IMPLS)
def test_workspace_contents_do_not_matter(pkg, cuda, name, impl):
    # every partial that the join reads was written by this call: NaN bytes stay unseen
    from conftest import import_module
    B, T, H, KVH, D, prefix, lengths, bs, counts = ATTENTION[name]
    d = make(B, T, H, KVH, D, torch.float16, prefix, lengths, bs, counts, scores=True)
    first = call(pkg, dict(d), cuda, impl)
    for key, buf in import_module("ops")._ws_cache.items():
        if key[2] == "shared_prefix":
            buf.fill_(0xff)
    again = call(pkg, dict(d), cuda, impl)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("D", [64, 128])
def test_pools_and_queries_at_any_address(pkg, cuda, D, dtype):
    # tensors that start one element into their storage: no 16-byte pieces, no TMA
    d = make(5, 3, 8, 2, D, dtype, 70, [3, 16, 17, 64, 90], scores=True)
    aligned = call(pkg, dict(d), cuda)
    moved = {}
    for n in ("q", "k", "v"):
        flat = torch.empty(d[n].numel() + 1, dtype=dtype, device=cuda)
        moved[n] = flat[1:].view(d[n].shape)
        moved[n].copy_(d[n])
    for names in (("q",), ("k", "v"), ("q", "k", "v")):
        out, sc = call(pkg, dict(d, **{n: moved[n] for n in names}), cuda)
        tol = 3e-3 if dtype == torch.float16 else 4e-5  # two results, each within its bound
        assert (out - aligned[0]).abs().max().item() <= tol
        torch.testing.assert_close(sc, aligned[1], rtol=4e-5, atol=4e-6)
    if dtype == torch.float16:
        with pytest.raises(RuntimeError, match="shape/alignment"):
            call(pkg, dict(d, k=moved["k"], v=moved["v"]), cuda, "mma")


def test_cells_past_two_to_the_31_elements(pkg, cuda):
    # pools of 4.3 GB: the last pages' cells lie past 2^31 elements
    KVH, D, bs = 8, 128, 16
    N = 2 ** 31 // (bs * KVH * D) + 64
    if torch.cuda.mem_get_info()[0] < 12 * N * bs * KVH * D:
        pytest.skip("needs 26 GB")
    k = torch.empty(N, bs, KVH, D, dtype=torch.float16, device=cuda)
    v = torch.empty_like(k)
    g = torch.Generator(device=cuda).manual_seed(3)
    for pool in (k, v):
        pool[-64:].normal_(generator=g)
        pool[:8].normal_(generator=g)
    q = torch.randn(2, 2, 32, D, generator=g, device=cuda).half()
    order = torch.randperm(60, device=cuda).to(torch.int32) + (N - 64)
    small = torch.arange(60, dtype=torch.int32, device=cuda)
    lengths = torch.tensor([150, 70], dtype=torch.int32, device=cuda)
    scores = torch.rand(2, KVH, 160, generator=g, device=cuda)
    ck, cv = k[order.long()].contiguous(), v[order.long()].contiguous()
    for impl in ("simt", "mma", "tcgen05"):
        far = pkg.shared_prefix_attention(q, k, v, order[:20], 310, order[20:40].view(2, 10), lengths,
                                          150, scores=scores, scores_out=torch.empty_like(scores),
                                          impl=impl_of(pkg, impl))
        near = pkg.shared_prefix_attention(q, ck, cv, small[:20], 310, small[20:40].view(2, 10),
                                           lengths, 150, scores=scores,
                                           scores_out=torch.empty_like(scores),
                                           impl=impl_of(pkg, impl))
        assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1])
    new = order[40:60].view(2, 10)
    kept, n, _ = pkg.evict_tokens(k, v, scores, order[20:40].view(2, 10), lengths, new, 100, 5)
    for b in range(2):
        for h in (0, KVH - 1):
            j = kept[b, h, :int(n[b])].long()
            src = order[20:40].view(2, 10)[b][j // bs].long()
            i = torch.arange(len(j), device=cuda)
            dst = new[b][i // bs].long()
            assert torch.equal(k[dst, i % bs, h], k[src, j % bs, h])
            assert torch.equal(v[dst, i % bs, h], v[src, j % bs, h])
    assert pkg.read_device_errors() == 0


def test_calls_on_two_streams_do_not_share_scratch(pkg, cuda):
    jobs = [make(20, 3, 8, 2, 64, torch.float16, 300, [5 + 3 * i for i in range(20)], seed=s)
            for s in range(2)]
    alone = [call(pkg, d, cuda) for d in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    inputs = [{n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()} for d in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, inputs)):
            with torch.cuda.stream(s):
                got[i].append(pkg.shared_prefix_attention(
                    c["q"], c["k"], c["v"], c["prefix_table"], c["prefix"], c["tables"],
                    c["lengths"], c["max_length"]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])


def test_scores_in_place_and_beside(pkg, cuda):
    d = make(3, 2, 8, 2, 64, torch.float16, 30, [4, 20, 67], scores=True)
    c = {n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()}
    args = (c["q"], c["k"], c["v"], c["prefix_table"], 30, c["tables"], c["lengths"], 67)
    beside = torch.full_like(c["scores"], float("nan"))
    out, same = pkg.shared_prefix_attention(*args, scores=c["scores"], scores_out=beside)
    assert same is beside and torch.equal(c["scores"].cpu(), d["scores"])
    out2, here = pkg.shared_prefix_attention(*args, scores=c["scores"])
    assert here is c["scores"] and torch.equal(here, beside) and torch.equal(out, out2)
    assert torch.equal(out, pkg.shared_prefix_attention(*args))


def test_attention_equals_paged_attention_without_a_prefix(pkg, cuda):
    d = make(5, 1, 8, 2, 128, torch.float16, 0, [1, 16, 17, 100, 300], stale=0.0)
    got = call(pkg, d, cuda)[:, 0]
    ref = pkg.paged_attention(d["q"][:, 0].contiguous().to(cuda), d["k"].to(cuda), d["v"].to(cuda),
                              d["tables"].to(cuda), d["lengths"].to(cuda), 300)
    assert (got - ref).abs().max().item() <= 2e-3


def test_three_dimensional_query_side_stream_and_graph(pkg, cuda):
    d = make(5, 1, 9, 3, 64, torch.float16, 100, [1, 16, 17, 100, 30])
    ref = call(pkg, d, cuda)
    c = {n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()}
    q = c["q"][:, 0].contiguous()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        def once():
            return pkg.shared_prefix_attention(q, c["k"], c["v"], c["prefix_table"], 100,
                                               c["tables"], c["lengths"], 100)
        got = once()
    s.synchronize()
    assert got.shape == q.shape and torch.equal(got, ref[:, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = once()
    held.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, ref[:, 0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_graph_replays_of_kernels_side_by_side(pkg, cuda, dtype):
    # a prefix kernel with the own-token kernel beside it, captured; the replays run
    # back to back, so that a call's partials are rewritten right after they were read
    d = make(24, 3, 8, 2, 64, dtype, 500, [3 + 11 * i for i in range(24)], scores=True)
    c = {n: t.to(cuda) if isinstance(t, torch.Tensor) else t for n, t in d.items()}
    beside = torch.empty_like(c["scores"])

    def once(q):
        return pkg.shared_prefix_attention(q, c["k"], c["v"], c["prefix_table"], 500, c["tables"],
                                           c["lengths"], d["max_length"], scores=c["scores"],
                                           scores_out=beside)[0]
    other = torch.randn_like(c["q"])
    want = [once(c["q"]).clone(), once(other).clone()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once(c["q"])
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = [once(q) for q in (c["q"], other) for _ in range(3)]
    for _ in range(5):
        for h in held:
            h.zero_()
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    for i, h in enumerate(held):
        assert torch.equal(h, want[i // 3])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_a_batch_past_the_lengths_kept_in_shared_memory(pkg, cuda, dtype):
    lengths = [(i * 37) % 41 for i in range(310)]
    check(pkg, make(310, 1, 2, 1, 64, dtype, 33, lengths, scores=True), cuda)


@pytest.mark.parametrize("impl", IMPLS)
def test_accumulated_weights_without_own_tokens(pkg, cuda, impl):
    d = make(2, 1, 4, 2, 64, torch.float16, 40, [0, 0], scores=True)
    out, sc = call(pkg, d, cuda, impl)
    assert torch.equal(sc.cpu(), d["scores"]) and torch.isfinite(out).all()


def test_given_output_at_any_address(pkg, cuda):
    d = make(3, 2, 8, 2, 64, torch.float16, 30, [4, 20, 67])
    want = call(pkg, d, cuda)
    flat = torch.empty(want.numel() + 1, dtype=torch.float16, device=cuda)
    for out in (torch.empty_like(want), flat[1:].view(want.shape)):
        assert call(pkg, d, cuda, out=out) is out and torch.equal(out, want)
    with pytest.raises(RuntimeError, match="invalid output tensor"):
        call(pkg, d, cuda, out=torch.empty_like(want, dtype=torch.float32))


def test_bad_metadata_is_flagged_not_followed(pkg, cuda):
    d = make(3, 2, 4, 2, 64, torch.float16, 40, [4, 20, 30], stale=0.0)
    for name, value, bit in (("lengths", [99, -4, 30], 0x2), ("counts", [3, -1, 2], 0x2),
                             ("tables", [[1 << 30] * 2] * 3, 0x1),
                             ("prefix_table", [-1, 10 ** 6, 0], 0x1)):
        e = dict(d, counts=torch.tensor([2, 2, 2], dtype=torch.int32))
        e[name] = torch.tensor(value, dtype=torch.int32)
        for impl in IMPLS:
            pkg.read_device_errors()
            out = call(pkg, e, cuda, impl)
            assert torch.isfinite(out).all()
            assert pkg.read_device_errors() & bit, (name, impl)


@pytest.mark.parametrize("what, message", [
    (dict(q="half strided"), "all tensors must be contiguous"),
    (dict(q=torch.zeros(3, 2, 4, 64, dtype=torch.bfloat16)), "use FP32 or FP16"),
    (dict(q=torch.zeros(3, 2, 5, 64).half()), "query heads must be a multiple of KV heads"),
    (dict(q=torch.zeros(3, 2, 4, 32).half()), "invalid cache shape"),
    (dict(q=torch.zeros(3, 2, 4, 64)), "dtype mismatch"),
    (dict(q=torch.zeros(3, 64).half()), "invalid Q/K/V shapes"),
    (dict(prefix=49), "invalid prefix length"),
    (dict(prefix=-1), "invalid prefix length"),
    (dict(max_length=33), "invalid context bound"),
    (dict(tables=torch.zeros(3, 2, dtype=torch.int64)), "metadata must be int32"),
    (dict(tables=torch.zeros(2, 2, dtype=torch.int32)), "invalid block tables"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), "invalid lengths"),
    (dict(counts=torch.zeros(3, dtype=torch.int64)), "invalid token counts"),
    (dict(scores=torch.zeros(3, 2, 29)), "scores must hold max_length tokens"),
    (dict(scores=torch.zeros(3, 4, 64)), "scores must be fp32"),
    (dict(scores=torch.zeros(3, 2, 64).half()), "scores must be fp32"),
])
def test_attention_refusals(pkg, cuda, what, message):
    d = make(3, 2, 4, 2, 64, torch.float16, 40, [4, 20, 30])
    if isinstance(what.get("q"), str):
        what = dict(q=d["q"].transpose(1, 2).contiguous().transpose(1, 2))
        with pytest.raises(RuntimeError, match=message):
            call(pkg, dict(d, q=what["q"].to(cuda)), cuda)
        return
    with pytest.raises(RuntimeError, match=message):
        call(pkg, dict(d, **what), cuda)


# ---- verification ------------------------------------------------------------
def drafts(B, T, V, dtype, seed=0, given=True, agree=0.5, lengths=None):
    g = torch.Generator().manual_seed(seed)
    target = torch.softmax(torch.randn(B, T + 1, V, generator=g) * 3, -1)
    draft = agree * target[:, :T] + (1 - agree) * torch.softmax(
        torch.randn(B, T, V, generator=g) * 3, -1)
    pick = draft if given else target[:, :T]
    tokens = torch.multinomial(pick.reshape(B * T, V), 1, generator=g).view(B, T)
    return dict(draft_tokens=tokens, target=target.to(dtype), draft=draft.to(dtype) if given else None,
                accept=torch.rand(B, T, generator=g), sample=torch.rand(B, generator=g),
                draft_lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32))


def verify(pkg, d, cuda):
    c = {n: t.to(cuda) if t is not None else None for n, t in d.items()}
    tokens, counts = pkg.verify_drafts(c["draft_tokens"], c["target"], c["accept"], c["sample"],
                                       draft_probs=c["draft"], draft_lengths=c["draft_lengths"])
    return tokens.cpu(), counts.cpu()


def check_verify(pkg, d, cuda):
    tokens, counts = verify(pkg, d, cuda)
    ref_tokens, ref_counts = oracle.verify_drafts(d["draft_tokens"], d["target"], d["accept"],
                                                  d["sample"], d["draft"], d["draft_lengths"])
    assert torch.equal(counts, ref_counts)
    assert torch.equal(tokens, ref_tokens)
    return tokens, counts


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("given", [True, False], ids=["draft probabilities", "looked up"])
@pytest.mark.parametrize("B, T, V", [(1, 1, 1), (1, 1, 2), (2, 3, 31), (5, 4, 129), (3, 8, 4096),
                                     (1, 3, 49152), (2, 2, 33001), (40, 2, 700), (2, 40, 64)])
def test_verify_drafts(pkg, cuda, B, T, V, given, dtype):
    for agree in (0.1, 0.9):
        check_verify(pkg, drafts(B, T, V, dtype, seed=B * 7 + T, given=given, agree=agree), cuda)


def test_verify_ragged_lengths(pkg, cuda):
    d = drafts(6, 5, 257, torch.float32, agree=0.95, lengths=[0, 5, 1, 3, 0, 4])
    tokens, counts = check_verify(pkg, d, cuda)
    assert (counts - 1 <= d["draft_lengths"]).all()
    assert pkg.read_device_errors() == 0


def test_verify_equal_distributions_accept_everything(pkg, cuda):
    d = drafts(8, 4, 500, torch.float32, agree=1.0)
    d["draft"] = d["target"][:, :4].clone()
    _, counts = check_verify(pkg, d, cuda)
    assert (counts == 5).all()


def test_verify_rows_whose_difference_leaves_nothing(pkg, cuda):
    # rejected (the draft has no target probability), but q >= p everywhere
    d = drafts(2, 2, 300, torch.float32)
    d["draft"] = (d["target"][:, :2] * 1.01)
    for b in range(2):
        d["target"][b, :, int(d["draft_tokens"][b, 0])] = 0.0
    _, counts = check_verify(pkg, d, cuda)
    assert (counts == 1).all()


def test_verify_without_any_weight(pkg, cuda):
    d = drafts(3, 2, 300, torch.float32)
    d["target"].zero_()
    tokens, counts = check_verify(pkg, d, cuda)
    assert (counts == 1).all() and (tokens == -1).all()


def test_verify_extreme_uniforms_and_values(pkg, cuda):
    d = drafts(7, 2, 1000, torch.float32)
    d["sample"] = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan"), 0.5])
    d["sample"][5] = 0.0
    check_verify(pkg, d, cuda)
    d = drafts(4, 2, 1000, torch.float32)
    d["target"][0, 0, ::3] = float("nan")
    d["target"][1, 0, 7] = float("inf")
    d["target"][2, 0, 5] = -1.0
    d["draft"][3, 0, 9] = float("nan")
    check_verify(pkg, d, cuda)


def test_verify_token_outside_the_vocabulary(pkg, cuda):
    for given in (True, False):
        d = drafts(3, 2, 100, torch.float32, given=given)
        d["draft_tokens"][0, 0], d["draft_tokens"][1, 0] = -5, 100
        pkg.read_device_errors()
        tokens, counts = verify(pkg, d, cuda)
        assert counts[0] == 1 and counts[1] == 1 and (tokens[:2, 0] >= 0).all()
        ref = oracle.verify_drafts(d["draft_tokens"], d["target"], d["accept"], d["sample"], d["draft"])
        assert torch.equal(tokens, ref[0]) and pkg.read_device_errors() == 0x40


def test_verify_refusals(pkg, cuda):
    good = drafts(2, 3, 50, torch.float32)
    for change, message in [
            (dict(target=good["target"][:, :3]), "invalid probabilities shape"),
            (dict(draft=good["draft"][:, :2]), "invalid probabilities shape"),
            (dict(draft=good["draft"].half()), "dtype mismatch"),
            (dict(target=good["target"].double()), "use FP32 or FP16"),
            (dict(draft_tokens=good["draft_tokens"].int()), "draft tokens must be int64"),
            (dict(accept=good["accept"].double()), "invalid random numbers"),
            (dict(sample=good["sample"][:1]), "invalid random numbers"),
            (dict(draft_lengths=torch.zeros(2, dtype=torch.int64)), "invalid draft lengths")]:
        d = dict(good, **change)
        d = {n: t.contiguous() if t is not None else None for n, t in d.items()}
        with pytest.raises(RuntimeError, match=message):
            verify(pkg, d, cuda)
    d = dict(good, target=good["target"].transpose(1, 2).contiguous().to(cuda).transpose(1, 2))
    with pytest.raises(RuntimeError, match="contiguous"):
        verify(pkg, d, cuda)


# ---- eviction ------------------------------------------------------------------
def cache(B, KVH, D, dtype, lengths, budget, bs=16, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    new = [-(-min(n, budget) // bs) for n in lengths]
    tables, rest, blocks = pages(lengths, bs, sum(new) + 2, g)
    new_tables = torch.zeros(B, max(1, -(-min(budget, max(max(lengths), 1) + extra) // bs)),
                             dtype=torch.int32)
    at = 0
    for b, n in enumerate(new):
        new_tables[b, :n] = rest[at:at + n]
        at += n
    return dict(k=torch.randn(blocks, bs, KVH, D, generator=g).to(dtype),
                v=torch.randn(blocks, bs, KVH, D, generator=g).to(dtype),
                scores=torch.randn(B, KVH, max(max(lengths), 1) + extra, generator=g).exp(),
                tables=tables, lengths=torch.tensor(lengths, dtype=torch.int32),
                new_tables=new_tables)


def check_evict(pkg, d, cuda, budget, recent):
    c = {n: t.to(cuda) for n, t in d.items()}
    kept, new_lengths, new_scores = pkg.evict_tokens(
        c["k"], c["v"], c["scores"], c["tables"], c["lengths"], c["new_tables"], budget, recent)
    ref = oracle.evict_tokens(d["scores"], d["lengths"], budget, recent)
    bs = d["k"].shape[1]
    k, v, s = d["k"].clone(), d["v"].clone(), torch.zeros_like(d["scores"])
    index = torch.full(kept.shape, -1, dtype=torch.int32)
    for b, row in enumerate(ref):
        assert int(new_lengths[b]) == min(int(d["lengths"][b]), budget)
        for h, keep in enumerate(row):
            for i, j in enumerate(keep):
                to, frm = int(d["new_tables"][b, i // bs]), int(d["tables"][b, j // bs])
                k[to, i % bs, h], v[to, i % bs, h] = d["k"][frm, j % bs, h], d["v"][frm, j % bs, h]
                s[b, h, i] = d["scores"][b, h, j]
                index[b, h, i] = j
    assert torch.equal(kept.cpu(), index)
    # copies: the same bits, NaN among them
    assert torch.equal(new_scores.cpu().view(torch.int32), s.view(torch.int32))
    assert torch.equal(c["k"].cpu(), k) and torch.equal(c["v"].cpu(), v)
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("B, KVH, D, lengths, budget, recent, bs", [
    (1, 1, 64, [1], 1, 0, 16), (1, 3, 64, [0], 4, 2, 16), (2, 2, 64, [5, 6], 5, 5, 16),
    (3, 2, 128, [16, 17, 64], 16, 4, 16), (4, 3, 64, [0, 1, 100, 333], 50, 7, 32),
    (2, 2, 64, [40, 30], 64, 8, 16), (2, 1, 7, [40, 90], 33, 8, 12), (2, 8, 128, [700, 300], 256, 0, 16),
    (1, 1, 64, [2048], 1000, 100, 16), (1, 2, 8, [5000], 4999, 0, 16), (1, 1, 8, [9000], 777, 50, 64),
])
def test_evict_tokens(pkg, cuda, B, KVH, D, lengths, budget, recent, bs, dtype):
    check_evict(pkg, cache(B, KVH, D, dtype, lengths, budget, bs), cuda, budget, recent)


def test_evict_ties_nan_infinities_and_zeros(pkg, cuda):
    d = cache(4, 2, 64, torch.float16, [200, 150, 90, 61], 60)
    d["scores"][0] = 0.0                                        # every score equal
    d["scores"][1, :, ::2] = float("nan")
    d["scores"][1, :, 1::4] = -float("inf")
    d["scores"][2, :, ::3] = float("inf")
    d["scores"][2, :, 1::3] = -0.0
    d["scores"][2, :, 2::3] = 0.0
    d["scores"][3] = -d["scores"][3]
    check_evict(pkg, d, cuda, 60, 10)


def test_evict_longer_than_one_round(pkg, cuda):
    d = cache(1, 1, 8, torch.float16, [20011], 6000, bs=64)
    d["scores"] = (d["scores"] * 4).floor()                     # many ties across rounds
    check_evict(pkg, d, cuda, 6000, 11)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_evict_rows_at_any_address(pkg, cuda, dtype):
    # few rows (copied by the selecting CTA) and many (by a kernel of their own)
    for lengths, budget, D in (([60, 90], 40, 64), ([700], 600, 128)):
        d = cache(len(lengths), 2, D, dtype, lengths, budget)
        c = {n: t.to(cuda) for n, t in d.items()}
        want = pkg.evict_tokens(c["k"], c["v"], c["scores"], c["tables"], c["lengths"],
                                c["new_tables"], budget, 3)
        moved = []
        for n in ("k", "v"):
            flat = torch.empty(d[n].numel() + 1, dtype=dtype, device=cuda)
            moved.append(flat[1:].view(d[n].shape))
            moved[-1].copy_(d[n])
        got = pkg.evict_tokens(*moved, c["scores"], c["tables"], c["lengths"], c["new_tables"],
                               budget, 3)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert torch.equal(moved[0], c["k"]) and torch.equal(moved[1], c["v"])


def test_evict_crowded_histogram_steps(pkg, cuda):
    # one outlier stretches the keys' range, so that all others share one step of the
    # histogram: more keys than are ranked, and more than are listed
    for n, budget in ((1200, 700), (6000, 2500), (20000, 9000)):
        d = cache(1, 2, 8, torch.float16, [n], budget, bs=64)
        g = torch.Generator().manual_seed(n)
        d["scores"] = 1.0 + torch.randint(0, 40, d["scores"].shape, generator=g) * 2.0 ** -23
        d["scores"][0, 0, 5], d["scores"][0, 1, 7] = 3e38, -3e38
        check_evict(pkg, d, cuda, budget, 11)


def test_evict_bad_metadata_is_flagged_not_followed(pkg, cuda):
    d = cache(2, 2, 64, torch.float16, [40, 60], 20)
    for name, value, bit in (("lengths", [-3, 1 << 20], 0x2), ("tables", [[1 << 28] * 4] * 2, 0x1),
                             ("new_tables", [[-7] * 2] * 2, 0x1)):
        e = dict(d)
        e[name] = torch.tensor(value, dtype=torch.int32)
        c = {n: t.to(cuda) for n, t in e.items()}
        pkg.read_device_errors()
        pkg.evict_tokens(c["k"], c["v"], c["scores"], c["tables"], c["lengths"], c["new_tables"], 20, 3)
        assert pkg.read_device_errors() & bit, name


def test_evict_refusals(pkg, cuda):
    d = cache(2, 2, 64, torch.float16, [40, 60], 20)
    for change, budget, recent, message in [
            (dict(), 0, 0, "invalid budget"), (dict(), 20, 21, "recent tokens must fit"),
            (dict(), 20, -1, "recent tokens must fit"), (dict(), 33, 0, "new tables must hold"),
            (dict(scores=d["scores"].double()), 20, 0, "scores must be fp32"),
            (dict(scores=d["scores"][:1].contiguous()), 20, 0, "scores must be fp32"),
            (dict(k=d["k"].float()), 20, 0, "dtype mismatch"),
            (dict(k=d["k"].double(), v=d["v"].double()), 20, 0, "use FP32 or FP16"),
            (dict(tables=d["tables"].long()), 20, 0, "metadata must be int32"),
            (dict(v=d["v"][:-1].contiguous()), 20, 0, "invalid cache shape")]:
        c = {n: t.to(cuda) for n, t in dict(d, **change).items()}
        with pytest.raises(RuntimeError, match=message):
            pkg.evict_tokens(c["k"], c["v"], c["scores"], c["tables"], c["lengths"],
                             c["new_tables"], budget, recent)
