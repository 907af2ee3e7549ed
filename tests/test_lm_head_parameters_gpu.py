"""An LM head and adapters that are parameters of a model in training."""
import pytest
import torch

from flashgen_b200.sampling.lm_head import AdapterHead

pytestmark = pytest.mark.gpu


def _param(*shape):
    return torch.nn.Parameter(torch.randn(*shape, device="cuda").half())


@pytest.mark.parametrize("dim", [64, 61])                 # used where it lies, laid out anew
def test_loading_parameters_builds_no_graph(cuda_device, dim):
    weight = _param(50, dim)
    head = AdapterHead(weight, slots=2, rank=8)
    for _ in range(3):
        down, up = _param(8, dim), _param(50, 8)
        head.load(1, down, up, 0.5)
        for bank in (head.weight, head._down, head._up, head._scales):
            assert not bank.requires_grad and bank.grad_fn is None
    hidden = torch.randn(3, dim, device="cuda").half()
    ids = torch.tensor([1, -1, 1], dtype=torch.int32, device="cuda")
    same = AdapterHead(weight.detach(), slots=2, rank=8)
    same.load(1, down.detach(), up.detach(), 0.5)
    assert torch.equal(head.logits(hidden, ids), same.logits(hidden, ids))
    assert down.grad is None and weight.requires_grad
