"""Host side of PrefixBatch (CPU): reservations, ids and refusals, on a runner without a model."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from conftest import import_module, import_pkg

KV = import_module("paged_kv")


class _Cfg:
    num_hidden_layers, num_key_value_heads, head_dim = 2, 2, 8
    num_attention_heads, hidden_size = 4, 32


def fake_runner(blocks=40, vocab=512, fail=None):
    cache = KV.DevicePagedKV(_Cfg, blocks=blocks, block_size=4, device="cpu", dtype=torch.float32,
                             max_batch=8, max_tokens=160)

    def prefill(ids, token_lists):
        if fail is not None:
            raise fail
        for rid, tokens in zip(ids, token_lists):
            cache.lengths[rid] = len(tokens)
    inner = SimpleNamespace(layers=[None] * 2, embed_tokens=SimpleNamespace(num_embeddings=vocab))
    return SimpleNamespace(cache=cache, prefill=prefill, device=torch.device("cpu"), heads=4, kv_heads=2,
                           head_dim=8, model=SimpleNamespace(model=inner))


@pytest.mark.parametrize("what, error", [
    (dict(prefix=[1] * 156), RuntimeError),                        # no pages for the prefix
    (dict(prefix=[1] * 20, max_own=80), RuntimeError),             # for one request, not for two
    (dict(prefix=[1] * 20, ids=["a", "b", "a"]), ValueError),      # an id twice
    (dict(prefix=[1] * 20, ids=["a", "taken"]), ValueError),       # somebody else's id
    (dict(prefix=[1] * 20, fail=RuntimeError("out of memory")), RuntimeError),
])
def test_a_group_that_cannot_be_set_up_keeps_no_pages(what, error):
    runner = fake_runner(fail=what.pop("fail", None))
    runner.cache.reserve("taken", 10)
    free, tables = sorted(runner.cache.free), dict(runner.cache.tables)
    a = dict(prefix=[1, 2], ids=["a", "b"], max_own=20)
    a.update(what)
    with pytest.raises(error):
        import_pkg().PrefixBatch(runner, a["prefix"], a["ids"], max_own=a["max_own"])
    assert sorted(runner.cache.free) == free and runner.cache.tables == tables


def test_groups_on_one_cache_have_their_own_prefix():
    runner = fake_runner()
    cache, pkg = runner.cache, import_pkg()
    one = pkg.PrefixBatch(runner, [1] * 10, ["a"], max_own=8)
    two = pkg.PrefixBatch(runner, [2] * 6, ["b"], max_own=8)
    none = pkg.PrefixBatch(runner, [], ["c"], max_own=8)
    assert one.prefix_table.numel() == 3 and two.prefix_table.numel() == 2
    assert none.prefix_table.numel() == 0 and none.prefix_length == 0
    assert not set(one.prefix_table.tolist()) & set(two.prefix_table.tolist())
    free = len(cache.free)
    none.close()  # a group without a prefix releases nobody's
    assert len(cache.free) == free + 2
    two.close()
    assert len(cache.free) == free + 6
    assert not set(one.prefix_table.tolist()) & set(cache.free)
    one.close()
    assert len(cache.free) == 40 and not cache.tables


def test_closing_twice_does_not_take_a_later_groups_requests():
    runner = fake_runner()
    first = import_pkg().PrefixBatch(runner, [1] * 10, ["a"], max_own=8)
    first.close()
    second = import_pkg().PrefixBatch(runner, [1] * 10, ["a"], max_own=8)
    free = len(runner.cache.free)
    first.close()
    assert len(runner.cache.free) == free and "a" in runner.cache.tables
    second.close()
    assert len(runner.cache.free) == 40


def test_a_budget_needs_pages_to_evict_into():
    # prefix 3 pages, two requests of 10; the budget needs 5 too
    pkg = import_pkg()
    runner = fake_runner(blocks=27)
    with pytest.raises(RuntimeError, match="no pages for the eviction"):
        pkg.PrefixBatch(runner, [1] * 10, ["a", "b"], max_own=40, budget=20, recent=4)
    assert len(runner.cache.free) == 27
    runner = fake_runner(blocks=28)
    batch = pkg.PrefixBatch(runner, [1] * 10, ["a", "b"], max_own=40, budget=20, recent=4)
    assert not runner.cache.free
    batch.close()
    assert len(runner.cache.free) == 28
    whole = fake_runner(blocks=23)  # nothing can pass this budget
    pkg.PrefixBatch(whole, [1] * 10, ["a", "b"], max_own=40, budget=40).close()
    with pytest.raises(ValueError, match="evicts nothing"):
        pkg.PrefixBatch(whole, [1] * 10, ["a", "b"], max_own=40).evict(["a"])


def unchanged(runner, batch, call, error=ValueError, match=None):
    before = dict(runner.cache.lengths), dict(batch.seen), sorted(runner.cache.free)
    with pytest.raises(error, match=match):
        call()
    assert before == (runner.cache.lengths, batch.seen, sorted(runner.cache.free))


def test_refusals_before_anything_is_computed():
    # the runner has no layers: a call that got further than its checks would fail otherwise
    runner = fake_runner(vocab=100)
    batch = import_pkg().PrefixBatch(runner, [1] * 10, ["a", "b"], max_own=8)
    for lists in ([[100], [1]], [[1], [-1]], [[1]], [[1], [2], [3]], [[], [1]], [[1] * 9, [1]]):
        unchanged(runner, batch, lambda: batch.score(lists))
    u, v = torch.rand(2, 3), torch.rand(2)
    good = dict(last=[1, 2], drafts=[[3, 4], []], u=u, v=v, temperature=1.0)

    def step(**kw):
        a = dict(good, **kw)
        return lambda: batch.step(a["last"], a["drafts"], a["u"], a["v"], temperature=a["temperature"])
    for kw, match in [
            (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
            (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
            (dict(drafts=[[1, 2, 3, 4], []]), "accept_uniforms"), (dict(drafts=[[3, 100], []]), "vocabulary"),
            (dict(drafts=[[-1], []]), "vocabulary"), (dict(last=[-1, 2]), "vocabulary"),
            (dict(last=[1]), "each request"), (dict(drafts=[[1]]), "each request"),
            (dict(u=torch.rand(3, 3)), "accept_uniforms"), (dict(u=torch.rand(2)), "accept_uniforms")]:
        unchanged(runner, batch, step(**kw), match=match)
    for prefix, kw in (([1, 100], {}), ([-1], {}), ([1], dict(budget=0, recent=0))):
        with pytest.raises(ValueError):
            import_pkg().PrefixBatch(runner, prefix, ["c"], max_own=8, **kw)
    batch.close()
    assert len(runner.cache.free) == 40
