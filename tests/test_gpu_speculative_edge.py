"""PrefixBatch where a step or a request goes other than planned: rejected drafts,
long prompts, full caches, failures in the middle. Set-up as in test_gpu_speculative.
"""
from __future__ import annotations

import pytest
import torch

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
