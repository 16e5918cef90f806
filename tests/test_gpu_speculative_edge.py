"""PrefixBatch where a step or a request goes other than planned: rejected drafts,
long prompts, full caches, failures in the middle. Set-up as in test_gpu_speculative.
"""
from __future__ import annotations

import pytest
import torch

from conftest import import_module
from test_gpu_speculative import setup

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
        assert runner.cache.lengths == other_runner.cache.lengths
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
