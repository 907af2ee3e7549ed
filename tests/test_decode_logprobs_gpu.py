"""The decode step from hidden states to ids with their log probabilities, and
the example that serves a mixed batch and moves one tenant's adapter."""
import importlib.util
import os

import pytest
import torch

from flashgen_b200 import AdapterHead, SamplingParams
from flashgen_b200.sampling.decode import DecodeBatch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _setup(B=9, dim=128, V=5003, slots=3):
    g = torch.Generator().manual_seed(0)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).cuda()

    weight = normal(V, dim, scale=3 * dim ** -0.5)
    head = AdapterHead(weight, slots=slots, rank=8)
    for s in range(slots):
        head.load(s, normal(8, dim, scale=dim ** -0.5), normal(V, 8, scale=0.3), 1.0)
    adapters = (torch.arange(B) % (slots + 1) - 1).to(torch.int32).cuda()
    params = [SamplingParams(temperature=0.9, top_k=40, repetition_penalty=1.1)] * B
    return head, adapters, params, normal, V


def test_step_hidden_reports_the_drawn_ids(cuda_device):
    head, adapters, params, normal, V = _setup()
    B = len(params)
    a, b = (DecodeBatch(params, V, capacity=16, device="cuda") for _ in range(2))
    total = torch.zeros(B, dtype=torch.float64)
    for step in range(4):
        hidden = normal(B, 128)
        u = torch.rand(B, device="cuda")
        logits = head.logits(hidden, adapters)
        plain = a.step(logits, uniforms=u).clone()                  # without log probabilities
        assert a.last_logprobs is None
        ids = b.step_hidden(hidden, head, adapters, uniforms=u, top_logprobs=4)
        assert torch.equal(ids, plain)                              # the ids do not depend on them
        r = b.last_logprobs
        lp = torch.log_softmax(logits.double(), 1).cpu()
        want = lp.gather(1, ids.cpu()[:, None])[:, 0]
        total += want
        # fp32 statistics over 5003 terms: below 1e-5 absolute on log probabilities below 30
        torch.testing.assert_close(r.logprobs.double().cpu(), want, atol=1e-5, rtol=0)
        torch.testing.assert_close(r.top_logprobs.double().cpu(), lp.topk(4, dim=1).values, atol=1e-5, rtol=0)
        assert (r.rank >= 0).all() and (r.rank < 40 + 16).all()     # drawn from the (penalised) top 40
    torch.testing.assert_close(b.cumulative_logprob.double().cpu(), total, atol=5e-5, rtol=0)
    assert b.histories() == a.histories()


def test_step_marks_rows_without_an_id(cuda_device):
    head, adapters, params, normal, V = _setup()
    dec = DecodeBatch(params, V, capacity=16, device="cuda")
    logits = head.logits(normal(len(params), 128), adapters).float()
    logits[2] = float("nan")
    logits[5] = -float("inf")
    ids = dec.step(logits, top_logprobs=2)
    assert ids[2] == -1 and ids[5] == -1
    r = dec.last_logprobs
    assert r.rank[2] == -1 and r.rank[5] == -1
    assert dec.cumulative_logprob[2] == 0 and dec.cumulative_logprob[5] == 0
    ok = [i for i in range(len(params)) if i not in (2, 5)]
    assert r.logprobs[ok].isfinite().all() and (r.logprobs[ok] < 0).all()


def test_example(cuda_device):
    spec = importlib.util.spec_from_file_location("adapter_policy_step",
                                                  os.path.join(ROOT, "examples", "adapter_policy_step.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main(requests=11, steps=4, dim=136, vocab=3001, slots=3)
    assert (r["served_logprob"] < 0).all() and r["served_logprob"].isfinite().all()
    assert r["after"] > r["before"]
