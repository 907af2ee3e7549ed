"""The block, the head, min-p sampling, log probabilities and clipping together, as a decode step
and a training step use them; and the example's gradients."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from flashgen_b200 import (AdapterHead, HeadBlock, SamplingParams, clip_grad_norm, fused_linear,
                           logprobs_and_entropy, sample_min_p)
from flashgen_b200.sampling.decode import DecodeBatch
from min_p_reference import sample_row

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16 = torch.bfloat16


def _parts(B=12, dim=96, V=3001, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(BF16).cuda()

    weight = normal(V, dim, scale=3 * dim ** -0.5)
    return normal, weight, HeadBlock(normal(dim, dim, scale=dim ** -0.5), normal(dim, scale=0.1))


def test_a_decode_step_from_hidden_states(cuda_device):
    B, V = 12, 3001
    normal, weight, block = _parts(B)
    head = AdapterHead(weight)
    params = [SamplingParams(temperature=0.8, min_p=[0.0, 0.05, 0.3][i % 3], top_p=0.95) for i in range(B)]
    dec = DecodeBatch(params, V, capacity=8, device="cuda", check_errors=True)
    for _ in range(3):
        hidden, u = normal(B, 96), torch.rand(B, device="cuda")
        ids = dec.step_hidden(hidden, head, block=block, out_dtype=torch.float32, uniforms=u, top_logprobs=2)
        logits = head.logits(fused_linear(hidden, block.weight, block.bias, hidden, activation="silu"),
                             out_dtype=torch.float32)
        x, us = logits.cpu().numpy(), u.cpu().numpy()
        for i in range(B):
            want = sample_row(x[i], us[i], params[i].min_p, 0.8, top_p=0.95)
            assert want.near or int(ids[i]) == want.id
        assert torch.equal(dec.last_logprobs.top_ids[:, 0], logits.argmax(1))


def test_a_policy_step(cuda_device):
    # draw, rescore under the model, back through the block, clip: against the same in 64 bits
    B, dim, V = 12, 96, 3001
    normal, weight, block = _parts(B, seed=1)
    x = normal(B, dim)
    leaves = [block.weight.clone().requires_grad_(), block.bias.clone().requires_grad_()]
    y = fused_linear(x, *leaves, x, activation="silu")
    with torch.no_grad():
        logits = AdapterHead(weight).logits(y, out_dtype=torch.float32)
        r = sample_min_p(logits, torch.rand(B, device="cuda"), torch.full((B,), 0.05, device="cuda"))
    assert (r.ids >= 0).all() and (r.logprobs <= 0).all()
    advantage = torch.linspace(-1, 1, B, device="cuda")
    logits.requires_grad_(True)
    lp, _ = logprobs_and_entropy(logits, r.ids)
    (advantage * lp).sum().backward()
    into_y = (logits.grad @ weight.float()).to(BF16)
    grads = list(torch.autograd.grad(y, leaves, into_y))
    before = [g.double() for g in grads]
    norm = clip_grad_norm(grads, 0.1)

    w64 = [t.detach().double().requires_grad_(True) for t in (block.weight, block.bias)]
    z = x.double() @ w64[0].T + w64[1]
    y64 = (z * torch.sigmoid(z) + x.double())
    # the head reads the block's rounded result; its gradient enters the block rounded
    lp64 = torch.log_softmax(y64.to(BF16).double() @ weight.double().T, 1).gather(1, r.ids[:, None])[:, 0]
    assert (lp.double() - lp64).abs().max() < 1e-4
    want = torch.autograd.grad(y64, w64, into_y.double())
    for g, e in zip(before, want):
        assert float((g - e).norm() / e.norm()) < torch.finfo(BF16).eps / 2
    total = float(torch.cat([g.flatten() for g in before]).norm())
    assert abs(float(norm) - total) <= 1e-6 * total
    for g, e in zip(grads, before):
        assert float((g.double() - e * 0.1 / total).norm()) <= torch.finfo(BF16).eps / 2 * 0.1


def test_a_captured_step(cuda_device):
    # block, head, draw and log probabilities in one graph, replayed on other inputs
    B, dim, V = 8, 96, 3001
    normal, weight, block = _parts(B, seed=2)
    head = AdapterHead(weight)
    x, u, mp = normal(B, dim), torch.rand(B, device="cuda"), torch.full((B,), 0.1, device="cuda")

    def step():
        logits = head.logits(block(x), out_dtype=torch.float32)
        return logits, sample_min_p(logits, u, mp)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, r = step()
    for seed in (3, 4):
        x.copy_(_parts(B, seed=seed)[0](B, dim))
        u.copy_(torch.rand(B, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        xs, us = logits.cpu().numpy(), u.cpu().numpy()
        for i in range(B):
            want = sample_row(xs[i], us[i], 0.1)
            assert want.near or (int(r.ids[i]), int(r.kept[i])) == (want.id, want.kept)


def test_the_example_clips_its_gradients(cuda_device):
    spec = importlib.util.spec_from_file_location("adapter_policy_step",
                                                  os.path.join(ROOT, "examples", "adapter_policy_step.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main(requests=11, steps=4, dim=136, vocab=3001, slots=3, limit=1e-3)
    assert np.isfinite(r["norm"]) and r["norm"] > 1e-3
    norm = float(torch.cat([g.double().flatten() for g in r["gradients"]]).norm())
    # fp32 gradients exactly, two bf16 ones to half a step
    assert abs(norm - 1e-3) <= 1e-3 * torch.finfo(BF16).eps / 2
