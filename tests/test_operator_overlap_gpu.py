"""Outputs that share memory with the inputs they are computed from, on the GPU."""
import pytest
import torch

from flashgen_b200 import AdapterHead, token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu


def test_gradient_and_its_logits(cuda_device):
    B, V = 7, 1000
    buf = torch.randn(B, 2 * V + 4, device="cuda")
    t = torch.randint(0, V, (B,), device="cuda")
    x = buf[:, :V]
    r = token_logprobs(x, t)
    ones = torch.ones(B, device="cuda")
    want = token_logprobs_grad(x, t, r.max, r.logsum, ones)
    for first in (1, 4, V - 1):
        with pytest.raises(RuntimeError, match="invalid argument"):
            token_logprobs_grad(x, t, r.max, r.logsum, ones, out=buf[:, first:first + V])
    with pytest.raises(RuntimeError, match="invalid argument"):                      # a row further
        token_logprobs_grad(x[:-1], t[:-1], r.max[:-1], r.logsum[:-1], ones[:-1], out=x[1:])
    assert torch.equal(token_logprobs_grad(x, t, r.max, r.logsum, ones, out=buf[:, V:2 * V]), want)   # beside it
    assert torch.equal(token_logprobs_grad(x, t, r.max, r.logsum, ones, out=x), want)                 # over it


def test_head_and_its_hidden_states(cuda_device):
    B, dim, V = 5, 64, 500
    head = AdapterHead(torch.randn(V, dim, device="cuda").half())
    buf = torch.randn(B, dim + V, device="cuda").half()
    want = head.logits(buf[:, :dim].clone())
    with pytest.raises(RuntimeError, match="invalid argument"):
        head.logits(buf[:, :dim], out=buf[:, dim - 1:dim - 1 + V])
    assert torch.equal(head.logits(buf[:, :dim], out=buf[:, dim:]), want)
