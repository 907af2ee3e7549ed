"""The norm that clipping returns holds its own four bytes, not the call's workspace."""
import pytest
import torch

from flashgen_b200 import clip_grad_norm, grad_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [1, 60, 700])
def test_a_kept_norm(cuda_device, count):
    grads = [torch.ones(5, device="cuda") for _ in range(count)]
    for norm in (grad_norm(grads), clip_grad_norm(grads, 1e9)):
        assert norm.shape == () and norm.untyped_storage().nbytes() == 4
    clip_grad_norm(grads, 1e9)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    kept = [clip_grad_norm(grads, 1e9) for _ in range(100)]
    assert torch.cuda.memory_allocated() - before <= 100 * 512          # the allocator's smallest blocks
    assert all(float(n) == float(kept[0]) for n in kept)
