"""What a head keeps of its weight: the weight itself where its rows are aligned, a snapshot otherwise."""
import pytest
import torch

from flashgen_b200.sampling.lm_head import AdapterHead

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,kept", [(64, True), (61, False)])
def test_updates_of_the_weight(cuda_device, dim, kept):
    weight = torch.randn(50, dim, device="cuda").half()
    head = AdapterHead(weight)
    hidden = torch.randn(3, dim, device="cuda").half()
    before = head.logits(hidden)
    assert (head.weight.data_ptr() == weight.data_ptr()) == kept
    weight.mul_(2)                                     # (a power of two: the logits double exactly)
    after = head.logits(hidden)
    assert torch.equal(after, before * 2 if kept else before)
    assert torch.equal(AdapterHead(weight).logits(hidden), before * 2)
