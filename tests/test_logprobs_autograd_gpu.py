"""The differentiable log probabilities in a graph, on the kernels."""
import pytest
import torch

from flashgen_b200 import SamplingParams
from flashgen_b200.sampling.decode import DecodeBatch
from flashgen_b200.sampling.lm_head import AdapterHead
from flashgen_b200.sampling.logprobs import logprobs_and_entropy, token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu


def _case(B=3, V=11):
    g = torch.Generator().manual_seed(0)
    return torch.randn(B, V, generator=g).cuda().requires_grad_(), torch.tensor([1, 2, 3])[:B].cuda()


@pytest.mark.parametrize("which", [0, 1])
def test_second_derivatives_are_refused(cuda_device, which):
    a, t = _case()
    out = logprobs_and_entropy(a * a, t)[which].sum()
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g,) = torch.autograd.grad(out, a, create_graph=True)
        torch.autograd.grad((g * g).sum(), a)


@pytest.mark.parametrize("change", ["index", "mul", "fill"])
def test_results_can_be_changed_in_place(cuda_device, change):
    """Masking padded tokens in place, as a trainer does first."""
    a, t = _case()
    keep = torch.tensor([1.0, 0.0, 1.0], device="cuda")
    lp, ent = logprobs_and_entropy(a, t)
    for v in (lp, ent):
        if change == "index":
            v[1] = 0
        elif change == "mul":
            v.mul_(keep)
        else:
            v.masked_fill_(keep == 0, 0.0)
    assert lp[1] == 0 and ent[1] == 0
    (lp.sum() + 0.5 * ent.sum()).backward()
    b = a.detach().clone().requires_grad_()
    z = torch.log_softmax(b, 1)
    (keep * (z.gather(1, t[:, None])[:, 0] - 0.5 * (z.exp() * z).sum(1))).sum().backward()
    torch.testing.assert_close(a.grad, b.grad, atol=2e-6, rtol=0)     # both in fp32 on terms below 4
    assert (a.grad[1] == 0).all()


def test_one_result_changed_leaves_the_other(cuda_device):
    """A detached result clamped for a report, and the statistics of a second call, change nothing saved."""
    a, t = _case()
    lp, ent = logprobs_and_entropy(a, t)
    lp.detach().clamp_(max=-5)
    ent.detach().zero_()
    ent.sum().backward()
    b = a.detach().clone().requires_grad_()
    z = torch.log_softmax(b, 1)
    (-(z.exp() * z).sum()).backward()
    torch.testing.assert_close(a.grad, b.grad, atol=2e-6, rtol=0)


def test_a_graph_notices_that_its_logits_were_written(cuda_device):
    a, t = _case()
    y = a * 1.0
    lp, _ = logprobs_and_entropy(y, t)
    r = token_logprobs(y.detach(), t)
    token_logprobs_grad(y.detach(), t, r.max, r.logsum, r.logprobs, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()
    head = AdapterHead(torch.randn(11, 64, device="cuda").half())
    y = (a * 1.0).half()
    lp, _ = logprobs_and_entropy(y, t)
    head.logits(torch.randn(3, 64, device="cuda").half(), out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()


def test_out_under_inference_mode(cuda_device):
    with torch.inference_mode():
        x = torch.randn(3, 11, device="cuda")
        r = token_logprobs(x)
        token_logprobs_grad(x, None, r.max, r.logsum, None, entropy=r.entropy, grad_entropy=r.entropy, out=x)
        head = AdapterHead(torch.randn(11, 64, device="cuda").half())
        head.logits(torch.randn(3, 64, device="cuda").half(), out=x)
    assert x.isfinite().all()


def test_gradients_that_do_not_exist_are_refused(cuda_device):
    a, t = _case()
    T = torch.ones(3, device="cuda").requires_grad_()
    with pytest.raises(RuntimeError, match="temperature"):
        logprobs_and_entropy(a, t, T)
    with torch.no_grad():
        logprobs_and_entropy(a, t, T)
    lp, _ = logprobs_and_entropy(a / T[:, None], t, None)              # the way that the error names
    lp.sum().backward()
    assert T.grad.isfinite().all() and (T.grad != 0).any()
    head = AdapterHead(torch.randn(11, 64, device="cuda").half())
    hidden = torch.randn(3, 64, device="cuda").half().requires_grad_()
    with pytest.raises(RuntimeError, match="backward"):
        head.logits(hidden)
    want = head.logits(hidden.detach())
    with torch.no_grad():
        assert torch.equal(head.logits(hidden), want)


def test_a_served_step_takes_hidden_states_that_require_gradients(cuda_device):
    head = AdapterHead(torch.randn(11, 64, device="cuda").half())
    hidden = torch.randn(3, 64, device="cuda").half()
    u = torch.full((3,), 0.5, device="cuda")
    ids = [DecodeBatch([SamplingParams()] * 3, 11, capacity=4).step_hidden(h, head, uniforms=u, top_logprobs=2).clone()
           for h in (hidden, hidden.clone().requires_grad_())]
    assert torch.equal(*ids)
