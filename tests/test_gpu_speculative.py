"""PrefixBatch (shared-prefix scoring, verification, eviction on a PagedLlama)
against the model's own dense forward pass, and the example's run.

Logit bar: as the runner's, 5e-3 of the largest logit in FP16 and 1e-5 in FP32 (the
two sides differ in the attention and RoPE kernels and in GEMM shapes).
"""
from __future__ import annotations

import subprocess
import sys

import pytest
import torch

import serving_oracle as oracle
from conftest import REPO
from oracle import llama_model as LM

pytestmark = pytest.mark.gpu


def setup(pkg, dtype, prefix_length=75, requests=3, **kw):
    model = LM.seeded_model(LM.tiny_llama_config(), 3, dtype, "cuda")
    runner = pkg.PagedLlama(model, blocks=256, block_size=16)
    g = torch.Generator().manual_seed(5)
    prefix = torch.randint(0, 512, (prefix_length,), generator=g).tolist()
    ids = list("abcdef"[:requests])
    return model, runner, prefix, ids, pkg.PrefixBatch(runner, prefix, ids, max_own=256, **kw), g


def dense(model, tokens):
    return model(torch.tensor([tokens], device="cuda")).logits[0].float()


@pytest.mark.parametrize("dtype, bar", [(torch.float16, 5e-3), (torch.float32, 1e-5)])
def test_scores_match_the_dense_model(pkg, cuda, dtype, bar):
    model, runner, prefix, ids, batch, g = setup(pkg, dtype)
    text = {r: [] for r in ids}
    for lengths in ([9, 1, 4], [1, 1, 1], [2, 5, 3]):
        lists = [torch.randint(0, 512, (n,), generator=g).tolist() for n in lengths]
        logits = batch.score(lists)
        for b, (r, tokens) in enumerate(zip(ids, lists)):
            text[r] += tokens
            want = dense(model, prefix + text[r])[-len(tokens):]
            err = (logits[b, :len(tokens)] - want).abs().max() / want.abs().max()
            assert err <= bar, (r, float(err))
    batch.close()
    assert pkg.read_device_errors() == 0


def test_step_verifies_and_rolls_back(pkg, cuda):
    model, runner, prefix, ids, batch, g = setup(pkg, torch.float32)
    text = {r: torch.randint(0, 512, (6,), generator=g).tolist() for r in ids}
    batch.score([text[r][:-1] for r in ids])
    for _ in range(5):
        drafts = []
        for b, r in enumerate(ids):  # some drafts are what the model finds likely, some are not
            guess, t = [], prefix + text[r]
            for i in range(3 - b):
                guess.append(int(dense(model, t)[-1].argmax()) if i < 2 else 7)
                t = t + guess[-1:]
            drafts.append(guess)
        u, v = torch.rand(3, 4, generator=g), torch.rand(3, generator=g)
        probs = torch.zeros(3, 5, 512)
        for b, r in enumerate(ids):
            n = len(drafts[b])
            p = torch.softmax(dense(model, prefix + text[r] + drafts[b])[-n - 1:] / 0.1, -1)
            probs[b, :n + 1] = p.cpu()
        want, counts = oracle.verify_drafts(
            torch.tensor([d + [0] * (4 - len(d)) for d in drafts]), probs, u, v,
            draft_lengths=torch.tensor([len(d) for d in drafts]))
        new = batch.step([text[r][-1] for r in ids], drafts, u.cuda(), v.cuda(), temperature=0.1)
        # the two sides' probabilities differ by rounding: a uniform that falls between
        # them would tell; none of these seeded ones does
        assert new == [w[:c] for w, c in zip(want.tolist(), counts.tolist())]
        for b, r in enumerate(ids):
            text[r] += new[b]
            assert runner.cache.lengths[r] == batch.seen[r] == len(text[r]) - 1
    batch.close()


def test_eviction_keeps_the_budget_and_a_wide_budget_changes_nothing(pkg, cuda):
    outputs = []
    for budget in (None, 200, 24):
        model, runner, prefix, ids, batch, g = setup(
            pkg, torch.float16, **({} if budget is None else dict(budget=budget, recent=8)))
        free = len(runner.cache.free)
        last = torch.randint(0, 512, (3,), generator=g).tolist()
        out = []
        for _ in range(20):
            u, v = torch.rand(3, 2, generator=g).cuda(), torch.rand(3, generator=g).cuda()
            new = batch.step(last, [[5, 9]] * 3, u, v)
            last = [n[-1] for n in new]
            out.append(new)
            if budget == 24:
                assert all(runner.cache.lengths[r] <= 24 for r in ids)
        outputs.append(out)
        assert len(runner.cache.free) == free  # pages swapped, none lost
        assert all(batch.seen[r] == sum(len(s[b]) for s in out) for b, r in enumerate(ids))
        if budget == 24:  # 20 tokens are there at least, and the cache is still used
            assert max(batch.seen.values()) >= 20
        batch.close()
    assert outputs[0] == outputs[1]
    assert pkg.read_device_errors() == 0


def test_accumulated_weights_sum_to_the_queries(pkg, cuda):
    # without a prefix every query row's weights sum to 1: each head of each real token
    model, runner, prefix, ids, batch, g = setup(pkg, torch.float32, prefix_length=0, budget=200)
    batch.score([[1, 2, 3], [4], [5, 6]])
    total = batch.scores.sum(-1)  # [layers, B, KVH]
    want = torch.tensor([3.0, 1.0, 2.0], device="cuda") * 2  # two query heads per kv head
    torch.testing.assert_close(total, want[None, :, None].expand_as(total), rtol=1e-5, atol=0)
    batch.close()


def test_arguments(pkg, cuda):
    model, runner, prefix, ids, batch, g = setup(pkg, torch.float16)
    with pytest.raises(ValueError):
        batch.score([[1], [], [2]])
    with pytest.raises(ValueError):
        batch.score([[1] * 257, [1], [2]])
    with pytest.raises(ValueError):
        pkg.PrefixBatch(runner, [1], ["x"], max_own=16, budget=32)
    batch.close()


def test_example_runs(cuda):
    r = subprocess.run([sys.executable, str(REPO / "examples" / "speculative_serving.py"), "--steps", "6"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "tokens in 6 steps of 8 requests" in r.stdout
