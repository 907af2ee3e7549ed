"""Clipping with an infinite limit scales and does no more, whatever the norm (a NaN one aside)."""
import math

import pytest
import torch

from flashgen_b200 import clip_grad_norm

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1.0, 0.5])
@pytest.mark.parametrize("shift", [0, 1])
def test_an_infinite_norm(cuda_device, dtype, scale, shift):
    base = torch.arange(1, 10001, device="cuda").remainder(97).to(dtype)       # halves are exact
    for bad in (math.inf, -math.inf):
        g = base.clone()[shift:]
        g[4321] = bad
        want = g * scale
        assert float(clip_grad_norm([g, base[:7].clone()], math.inf, scale=scale)) == math.inf
        assert torch.equal(g, want)
    g = base.clone()[shift:]
    g[17] = math.nan
    assert math.isnan(float(clip_grad_norm(g, math.inf, scale=scale))) and g.isnan().all()


def test_finite_gradients_of_an_infinite_norm(cuda_device):
    g = torch.full((1000,), 2.0 ** 127, device="cuda")
    want = g * 0.25
    out = torch.empty_like(g)
    assert float(clip_grad_norm(g, math.inf, scale=0.25, out=out)) == math.inf
    assert torch.equal(out, want)
    assert float(clip_grad_norm(g, 1.0)) == math.inf and (g == 0).all()
