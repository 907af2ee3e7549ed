"""The differentiable log probabilities in a graph, on the kernels."""
import pytest
import torch

from flashgen_b200.sampling.logprobs import logprobs_and_entropy

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
