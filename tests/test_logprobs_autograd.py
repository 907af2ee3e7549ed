"""What autograd sees of the token log probabilities, with torch operations in the place of the two
kernels (no GPU)."""
import pytest
import torch

from flashgen_b200.sampling import logprobs as L


def _forward(logits, tokens=None, *, temperature=None, top=0, check_errors=False):
    T = torch.ones(len(logits)) if temperature is None else temperature
    y = (logits - logits.max(dim=1, keepdim=True).values) / T[:, None]
    lp = torch.log_softmax(y, 1)
    own = torch.stack([lp.gather(1, tokens[:, None])[:, 0], -(lp.exp() * lp).sum(1), logits.max(dim=1).values,
                       y.exp().sum(1).log()])
    return L.TokenLogprobs(*own.clone().unbind(0), None, None, None, None)


def _backward(logits, tokens, max, logsum, grad_logprobs, *, entropy=None, grad_entropy=None, temperature=None, out=None):
    T = torch.ones(len(logits)) if temperature is None else temperature
    lp = (logits - max[:, None]) / T[:, None] - logsum[:, None]
    p = lp.exp()
    d = torch.zeros_like(logits)
    if grad_logprobs is not None:
        d = d - grad_logprobs[:, None] * p
        d = d.scatter_add(1, tokens[:, None], grad_logprobs[:, None])
    if grad_entropy is not None:
        d = d - grad_entropy[:, None] * p * (lp + entropy[:, None])
    return d / T[:, None]


@pytest.fixture
def stand_ins(monkeypatch):
    monkeypatch.setattr(L, "token_logprobs", _forward)
    monkeypatch.setattr(L, "token_logprobs_grad", _backward)


def _case(B=3, V=11):
    g = torch.Generator().manual_seed(0)
    return torch.randn(B, V, generator=g).requires_grad_(), torch.tensor([1, 2, 3])[:B]


def test_first_derivatives(stand_ins):
    a, t = _case()
    lp, ent = L.logprobs_and_entropy(a * a, t)
    (got,) = torch.autograd.grad(lp.sum() + ent.sum(), a)
    z = torch.log_softmax(a * a, 1)
    (want,) = torch.autograd.grad(z.gather(1, t[:, None]).sum() - (z.exp() * z).sum(), a)
    torch.testing.assert_close(got, want, atol=1e-5, rtol=0)


@pytest.mark.parametrize("which", [0, 1])
def test_second_derivatives_are_refused(stand_ins, which):
    """There is no second derivative: a penalty on gradients must not lose its term without a word."""
    a, t = _case()
    out = L.logprobs_and_entropy(a * a, t)[which].sum()
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g,) = torch.autograd.grad(out, a, create_graph=True)
        torch.autograd.grad((g * g).sum(), a)


def test_a_graph_that_is_not_used_again(stand_ins):
    """create_graph=True alone, for the rest of a loss, is no second derivative of these terms."""
    a, t = _case()
    lp, _ = L.logprobs_and_entropy(a, t)
    (g,) = torch.autograd.grad(lp.sum() + (a ** 3).sum(), a, create_graph=True)
    z = torch.log_softmax(a, 1).gather(1, t[:, None]).sum() + (a ** 3).sum()
    (want,) = torch.autograd.grad(z, a)
    torch.testing.assert_close(g.detach(), want, atol=1e-5, rtol=0)


def test_a_learned_temperature_is_refused(stand_ins):
    a, t = _case()
    T = torch.ones(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="temperature"):
        L.logprobs_and_entropy(a, t, T)
    lp, _ = L.logprobs_and_entropy(a, t, T.detach())
    lp.sum().backward()
    assert a.grad.isfinite().all()
