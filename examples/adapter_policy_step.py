"""A policy-gradient step on one tenant's adapter while a mixed batch is served.

1. Requests of several tenants decode together: one LM head, every row with its
   own low-rank adapter, ids drawn by the fused sampler, log probabilities and
   alternatives reported (``DecodeBatch.step_hidden``).
2. The rollouts of one tenant are rescored with gradients
   (``logprobs_and_entropy``) and its adapter's ``up`` matrix takes one step
   that raises the reward's expectation.

The hidden states stand in for a model's last layer: random rows, one per
request and step.

    python examples/adapter_policy_step.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from flashgen_b200 import AdapterHead, SamplingParams, logprobs_and_entropy  # noqa: E402
from flashgen_b200.sampling.decode import DecodeBatch  # noqa: E402


def main(requests: int = 24, steps: int = 8, dim: int = 512, vocab: int = 32000, slots: int = 4, rank: int = 8,
         rate: float = 20.0, device: str = "cuda", seed: int = 0) -> dict:
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, scale):
        return (torch.randn(shape, device=device, generator=gen) * scale).to(torch.bfloat16)

    head = AdapterHead(normal(vocab, dim, scale=2 * dim ** -0.5), slots=slots, rank=rank)
    down = [normal(rank, dim, scale=dim ** -0.5) for _ in range(slots)]
    up = [normal(vocab, rank, scale=0.05) for _ in range(slots)]
    for s in range(slots):
        head.load(s, down[s], up[s])
    adapters = (torch.arange(requests, device=device) % (slots + 1) - 1).to(torch.int32)   # -1: no adapter

    # ---- serve: decode the mixed batch, with log probabilities ----
    batch = DecodeBatch([SamplingParams(temperature=0.8, top_k=50, repetition_penalty=1.05)] * requests, vocab,
                        capacity=64, device=device)
    hidden, tokens = [], []
    for _ in range(steps):
        h = normal(requests, dim, scale=1.0)
        ids = batch.step_hidden(h, head, adapters, top_logprobs=3, generator=gen)
        hidden.append(h)
        tokens.append(ids.clone())
    served = batch.cumulative_logprob.clone()

    # ---- train: rescore tenant 0's rollouts and move its adapter ----
    mine = torch.nonzero(adapters == 0)[:, 0]
    x = torch.cat([h[mine] for h in hidden])
    t = torch.cat([ids[mine] for ids in tokens])
    reward = (t < vocab // 2).float()                       # this tenant wants small ids
    advantage = (reward - reward.mean()) / t.numel()

    def objective(b: torch.Tensor, grad: bool):
        head.load(0, down[0], b)
        logits = head.logits(x, torch.zeros(len(x), dtype=torch.int32, device=device), out_dtype=torch.float32)
        logits.requires_grad_(grad)
        logprobs, entropy = logprobs_and_entropy(logits, t)
        value = (advantage * logprobs).sum() + 1e-4 * entropy.mean()
        return value, logits

    before, logits = objective(up[0], True)
    before.backward()
    u = x.float() @ down[0].float().T                       # d logits / d up = U^T
    up[0] = (up[0].float() + rate * logits.grad.T @ u).to(torch.bfloat16)
    after, _ = objective(up[0], False)
    return {"served_logprob": served, "last": batch.last_logprobs, "before": float(before.detach()),
            "after": float(after)}


if __name__ == "__main__":
    r = main()
    print("cumulative log probability of the served rows:", [round(v, 2) for v in r["served_logprob"].tolist()])
    print("alternatives of row 0 at the last step:", r["last"].top_ids[0].tolist(),
          [round(v, 3) for v in r["last"].top_logprobs[0].tolist()])
    print(f"objective of tenant 0: {r['before']:.4f} -> {r['after']:.4f}")
