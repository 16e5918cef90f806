"""Requests that share an instruction prefix, decoded speculatively on a bounded cache.

Drafts are looked up in each request's own text (the tokens that followed the
latest earlier occurrence of its last token), so no draft model is needed. The
model is a randomly initialised Llama: what it says means nothing, what runs is
the path a served model takes.

    python examples/speculative_serving.py [--requests 8] [--steps 24] [--drafts 4]
"""
import argparse
import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
b200 = importlib.import_module("distributed-llm-inference_b200")


def look_up(text, drafts):
    """The tokens after the latest earlier occurrence of the last one."""
    for at in range(len(text) - 2, -1, -1):
        if text[at] == text[-1]:
            return text[at + 1:at + 1 + drafts]
    return []


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--requests", type=int, default=8)
    parser.add_argument("--steps", type=int, default=24)
    parser.add_argument("--drafts", type=int, default=4)
    parser.add_argument("--budget", type=int, default=32)
    args = parser.parse_args()
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    config = LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                         num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                         tie_word_embeddings=True)
    model = LlamaForCausalLM(config).half().cuda()
    runner = b200.PagedLlama(model, blocks=1024, block_size=16)
    g = torch.Generator().manual_seed(1)
    prefix = torch.randint(0, 512, (300,), generator=g).tolist()
    ids = [f"request {i}" for i in range(args.requests)]
    text = {rid: torch.randint(0, 512, (12,), generator=g).tolist() for rid in ids}
    batch = b200.PrefixBatch(runner, prefix, ids, max_own=512, budget=args.budget, recent=16)
    # the requests' own prompts, all but the last token; their logits are not needed
    batch.score([text[rid][:-1] for rid in ids], last_only=True)
    made = 0
    for _ in range(args.steps):
        drafts = [look_up(text[rid], args.drafts) for rid in ids]
        new = batch.step([text[rid][-1] for rid in ids], drafts,
                         torch.rand(args.requests, args.drafts, device="cuda"),
                         torch.rand(args.requests, device="cuda"), temperature=0.3)
        for rid, tokens in zip(ids, new):
            text[rid] += tokens
            made += len(tokens)
    print(f"{made} tokens in {args.steps} steps of {args.requests} requests; own tokens cached: "
          f"{[runner.cache.lengths[rid] for rid in ids]} of {[batch.seen[rid] for rid in ids]} seen")
    batch.close()


if __name__ == "__main__":
    main()
