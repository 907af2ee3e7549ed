"""The fused linear block's gradients under hooks on saved tensors: offloading and cloning
bring a slice of a wider buffer back dense; the gradients are the same bits."""
import pytest
import torch

from flashgen_b200 import fused_linear
from test_linear_gpu import BF16, F16, tensors

pytestmark = pytest.mark.gpu


def hooks(kind):
    if kind == "cpu":
        return torch.autograd.graph.save_on_cpu(pin_memory=True)
    if kind == "clone":
        return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)
    # unaligned: every tensor comes back two elements into a buffer
    def away(t):
        flat = torch.empty(t.numel() + 2, dtype=t.dtype, device=t.device)[2:]
        flat.copy_(t.reshape(-1))
        return flat.view(t.shape)
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, away)


@pytest.mark.parametrize("kind", ["cpu", "clone", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("size", [(50, 72, 88), (1, 72, 88), (50, 77, 91), (300, 256, 128)])
@pytest.mark.parametrize("lo", [0, 3])
def test_hooks(cuda_device, kind, dtype, act, size, lo):
    tokens, inner, outer = size
    x, w, b, r, gy = tensors(*size, dtype, seed=21)
    wide = [torch.full((t.shape[0], inner + 32 + lo), float("nan"), dtype=dtype, device="cuda") for t in (x, w)]
    for buf, t in zip(wide, (x, w)):
        buf[:, lo:lo + inner] = t
    leaves = [wide[0][:, lo:lo + inner].requires_grad_(), wide[1][:, lo:lo + inner].requires_grad_(), b.requires_grad_()]
    want = torch.autograd.grad(fused_linear(*leaves, r, activation=act), leaves, gy)
    with hooks(kind):
        out = fused_linear(*leaves, r, activation=act)
    got = torch.autograd.grad(out, leaves, gy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert not any(g.isnan().any() for g in got)


@pytest.mark.parametrize("inner", [72, 77])
def test_recomputed(cuda_device, inner):
    # a block that is computed again in the backward pass instead of being kept
    from torch.utils.checkpoint import checkpoint
    x, w, b, r, gy = tensors(50, inner, 88, BF16, seed=22)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def block(x, w, b):
        return fused_linear(x * 2, w, b, r, activation="gelu")

    want = torch.autograd.grad(block(*leaves), leaves, gy)
    got = torch.autograd.grad(checkpoint(block, *leaves, use_reentrant=False), leaves, gy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
