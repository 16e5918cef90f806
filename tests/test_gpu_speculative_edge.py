"""PrefixBatch where a step or a request goes other than planned: rejected drafts,
long prompts, full caches, failures in the middle. Set-up as in test_gpu_speculative.
"""
from __future__ import annotations

import pytest
import torch

from conftest import import_module
from oracle import llama_model as LM
from test_gpu_speculative import dense, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("accepted", [0, 1, 3])
def test_rejected_drafts_leave_no_weight(pkg, cuda, accepted):
    # u = 0 accepts a draft that was not sampled (0 < p), u = 1 rejects it
    drafts = [[5, 9, 7], [1, 2, 3], [11, 400, 8]]
    _, runner, _, ids, batch, g = setup(pkg, torch.float32, budget=200)
    _, other_runner, _, _, other, _ = setup(pkg, torch.float32, budget=200)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (6, 1, 9)]
    batch.score(prompts)
    other.score(prompts)
    u = torch.ones(3, 3)
    u[:, :accepted] = 0.0
    for last in ([3, 4, 5], [100, 101, 102]):
        new = batch.step(last, drafts, u.cuda(), torch.full((3,), 0.5).cuda())
        assert [n[:-1] for n in new] == [d[:accepted] for d in drafts]
        other.score([[a, *d[:accepted]] for a, d in zip(last, drafts)])
        assert all(runner.cache.lengths[r] == other_runner.cache.lengths[r] for r in "abc")
        # the same FP32 sums in another order: 2e-5 of a weight each, as the operator's own bound
        torch.testing.assert_close(batch.scores, other.scores, rtol=4e-5, atol=4e-6)
    total = batch.scores.sum(-1)  # prefix of 75 tokens: own tokens get part of each row's 1
    assert (total > 0).all()
    batch.close()
    other.close()
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("where", ["score", "step", "weights", "eviction"])
def test_a_failure_in_the_middle_changes_nothing(pkg, cuda, where, monkeypatch):
    module = import_module("speculative")
    batches = [setup(pkg, torch.float32, budget=16, recent=4) for _ in range(2)]
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (14, 2, 9)]
    for _, _, _, _, batch, _ in batches:
        batch.score(prompts)
    (_, runner, _, ids, batch, _), twin = batches[0], batches[1][4]
    u, v = torch.zeros(3, 2, device=cuda), torch.full((3,), 0.3, device=cuda)
    before = (dict(runner.cache.lengths), {r: list(t) for r, t in runner.cache.tables.items()},
              sorted(runner.cache.free), dict(batch.seen), batch.scores.clone())
    name = "evict_tokens" if where == "eviction" else "shared_prefix_attention"
    left = [3 if where == "weights" else 1]  # two layers: the third call is the weights' first
    real = getattr(module, name)

    def failing(*args, **kw):
        left[0] -= 1
        if left[0] < 0:
            raise RuntimeError("out of memory")
        return real(*args, **kw)
    with monkeypatch.context() as m:
        m.setattr(module, name, failing)
        with pytest.raises(RuntimeError, match="out of memory"):
            if where == "score":
                batch.score([[7], [8, 9], [10]])
            else:
                batch.step([7, 8, 9], [[1, 2]] * 3, u, v)
    assert before[0] == runner.cache.lengths and before[3] == batch.seen
    assert before[1] == runner.cache.tables and before[2] == sorted(runner.cache.free)
    assert torch.equal(before[4], batch.scores)
    for _ in range(2):  # the same calls go on as in a batch where nothing failed
        assert batch.step([7, 8, 9], [[1, 2]] * 3, u, v) == twin.step([7, 8, 9], [[1, 2]] * 3, u, v)
        assert batch.seen == twin.seen and torch.equal(batch.scores, twin.scores)
    assert max(runner.cache.lengths[r] for r in ids) <= 16
    batch.close()
    twin.close()
    assert pkg.read_device_errors() == 0


def test_long_runs_are_scored_in_pieces(pkg, cuda, monkeypatch):
    # logits, weights and steps as without pieces; no call takes more scratch than it may
    module = import_module("speculative")
    batches = [setup(pkg, torch.float32, budget=128, recent=8) for _ in range(2)]
    (model, _, prefix, ids, batch, g), twin = batches[0], batches[1][4]
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (120, 1, 47)]
    drafts = [[3, 7, 5, 6, 2, 9], [8], []]
    u, v = torch.zeros(3, 6, device=cuda), torch.full((3,), 0.7, device=cuda)
    u[0, 4:] = 1.0  # four of six accepted
    want = twin.score(prompts), twin.step([1, 2, 3], drafts, u, v)
    sizes, real = [], module.shared_prefix_attention

    def measured(q, *args, **kw):
        out = real(q, *args, **kw)
        scored = args[6] if kw.get("scores") is not None else 0
        sizes.append((q.shape[1], 4 * q.shape[0] * q.shape[1] * q.shape[2] * (2 * q.shape[3] + scored)))
        return out
    limit = 4 * 3 * 4 * (2 * 64 + 130) * 3  # three tokens of 3 requests with 4 heads of 64
    monkeypatch.setattr(module, "_SCRATCH", limit, raising=False)
    monkeypatch.setattr(module, "shared_prefix_attention", measured)
    got = batch.score(prompts)
    assert max(size for _, size in sizes) <= limit and max(t for t, _ in sizes) > 1
    for b, (rid, tokens) in enumerate(zip(ids, prompts)):
        ref = dense(model, prefix + tokens)[-len(tokens):]
        for logits in (got, want[0]):  # the runner's own bar
            assert (logits[b, :len(tokens)] - ref).abs().max() <= 1e-5 * ref.abs().max()
    assert batch.step([1, 2, 3], drafts, u, v) == want[1]
    assert max(size for _, size in sizes) <= limit
    assert batch.seen == twin.seen
    torch.testing.assert_close(batch.scores, twin.scores, rtol=4e-5, atol=4e-6)
    batch.close()
    twin.close()


def test_a_prompt_past_one_calls_tokens(pkg, cuda):
    model = LM.seeded_model(LM.tiny_llama_config(), 3, torch.float32, "cuda")
    runner = pkg.PagedLlama(model, blocks=300, block_size=16)
    batch = pkg.PrefixBatch(runner, [5, 6, 7], ["a"], max_own=4300)
    prompt = torch.randint(0, 512, (4200,), generator=torch.Generator().manual_seed(2)).tolist()
    got, want = batch.score([prompt])[0], dense(model, [5, 6, 7] + prompt)[-4200:]
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    batch.close()


def test_a_full_cache_still_evicts(pkg, cuda):
    # no free pages but those in reserve: the same tokens, scores and lengths as with room
    prefix = torch.randint(0, 512, (75,), generator=torch.Generator().manual_seed(5)).tolist()
    results = []
    for spare in (0, 2, 300):  # pages beyond the prefix's 5, the requests' 3 x 6 and the reserve's 2
        model = LM.seeded_model(LM.tiny_llama_config(), 3, torch.float32, "cuda")
        runner = pkg.PagedLlama(model, blocks=5 + 18 + 2 + spare, block_size=16)
        batch = pkg.PrefixBatch(runner, prefix, ["a", "b", "c"], max_own=90, budget=24, recent=8)
        free = len(runner.cache.free)
        assert free == spare
        g = torch.Generator().manual_seed(1)
        last, out = [1, 2, 3], []
        for _ in range(25):
            u, v = torch.rand(3, 3, generator=g).cuda(), torch.rand(3, generator=g).cuda()
            new = batch.step(last, [[5, 9, 11]] * 3, u, v)
            last = [n[-1] for n in new]
            out.append((new, batch.scores.clone()))
            assert max(runner.cache.lengths[r] for r in "abc") <= 24
            pages = [p for t in runner.cache.tables.values() for p in t] + runner.cache.free
            assert sorted(pages) == list(range(runner.cache.total_blocks))  # each in one place
            assert [len(runner.cache.tables[r]) for r in "abc"] == [6, 6, 6]
            assert len(runner.cache.free) == free
        results.append(out)
        batch.close()
        assert len(runner.cache.free) == runner.cache.total_blocks
    for other in results[1:]:
        for (new, scores), (new2, scores2) in zip(results[0], other):
            assert new == new2 and torch.equal(scores, scores2)
    assert pkg.read_device_errors() == 0


def test_a_later_cut_that_fails_waits_for_the_next_step(pkg, cuda, monkeypatch):
    module = import_module("speculative")
    prefix = [4] * 20
    batches = []
    for _ in range(2):
        model = LM.seeded_model(LM.tiny_llama_config(), 3, torch.float32, "cuda")
        runner = pkg.PagedLlama(model, blocks=2 + 6 + 1, block_size=16)
        batches.append(pkg.PrefixBatch(runner, prefix, ["a", "b"], max_own=40, budget=16, recent=4))
        batches[-1].score([[i % 7 for i in range(15)], [i % 5 for i in range(15)]])
    batch, twin = batches
    u, v = torch.zeros(2, 2, device=cuda), torch.full((2,), 0.3, device=cuda)
    real, left = module.evict_tokens, [2]  # two layers of the first request

    def failing(*args):
        left[0] -= 1
        if left[0] < 0:
            raise RuntimeError("out of memory")
        return real(*args)
    with monkeypatch.context() as m:
        m.setattr(module, "evict_tokens", failing)
        with pytest.warns(UserWarning, match="over their budget"):
            got = batch.step([7, 8], [[1, 2]] * 2, u, v)
    assert got == twin.step([7, 8], [[1, 2]] * 2, u, v)
    assert batch.runner.cache.lengths["a"] == 16 and batch.runner.cache.lengths["b"] == 18
    assert batch.seen == twin.seen and torch.equal(batch.scores[:, 0], twin.scores[:, 0])
    batch.evict(["b"])
    assert batch.runner.cache.lengths["b"] == 16 and torch.equal(batch.scores, twin.scores)
    assert batch.step([7, 8], [[1, 2]] * 2, u, v) == twin.step([7, 8], [[1, 2]] * 2, u, v)


def test_logits_that_are_not_numbers_end_the_step(pkg, cuda, monkeypatch):
    _, runner, _, ids, batch, g = setup(pkg, torch.float32, budget=64, recent=8)
    batch.score([[1, 2], [3], [4, 5, 6]])
    before = dict(runner.cache.lengths), dict(batch.seen), batch.scores.clone()
    u, v = torch.rand(3, 2, generator=g).cuda(), torch.rand(3, generator=g).cuda()
    head = runner.model.lm_head
    nan = torch.nn.Module()
    nan.forward = lambda x: head(x) * float("nan")
    monkeypatch.setattr(runner.model, "lm_head", nan)
    with pytest.raises(RuntimeError, match="no token to draw"):
        batch.step([7, 8, 9], [[1, 2], [], [3]], u, v)
    assert before[:2] == (runner.cache.lengths, batch.seen) and torch.equal(before[2], batch.scores)
    monkeypatch.setattr(runner.model, "lm_head", head)
    new = batch.step([7, 8, 9], [[1, 2], [], [3]], u, v)
    assert all(0 <= t < 512 for got in new for t in got)
    batch.close()
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("pieces", [False, True])
def test_last_logits_alone(pkg, cuda, pieces, monkeypatch):
    batches = [setup(pkg, torch.float32, budget=128, recent=8) for _ in range(2)]
    (_, runner, _, _, batch, g), twin = batches[0], batches[1][4]
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (50, 1, 47)]
    want = twin.score(prompts)
    if pieces:
        monkeypatch.setattr(import_module("speculative"), "_SCRATCH", 4 * 3 * 4 * (2 * 64 + 60) * 7)
    rows = []
    hook = runner.model.lm_head.register_forward_pre_hook(lambda m, a: rows.append(a[0].shape[:-1].numel()))
    got = batch.score(prompts, last_only=True)
    hook.remove()
    assert rows == [3] and got.shape == (3, 512) and got.dtype == torch.float32
    last = torch.stack([want[b, len(p) - 1] for b, p in enumerate(prompts)])
    # both within the runner's own bar of the dense model
    assert (got - last).abs().max() <= 2e-5 * last.abs().max()
    assert batch.seen == twin.seen
    torch.testing.assert_close(batch.scores, twin.scores, rtol=4e-5, atol=4e-6)
    batch.close()
    twin.close()
