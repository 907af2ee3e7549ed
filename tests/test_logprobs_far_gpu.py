"""Token log probabilities and their gradient where logits lie far from 0 in units of the temperature:
masks of every size between -1e4 and the type's lowest value, rows far from 0 as a whole, and rows on
both sides of the distance from which a row is summed by differences. The bounds are those of
tests/logprob_reference.py: nothing in them depends on how far from 0 a row lies."""
import math

import pytest
import torch

from tests.test_logprobs_gpu import DTYPES, _check, _grad_case

pytestmark = pytest.mark.gpu
SHAPES = [(1, 50257), (4, 5000), (300, 2309)]   # a cluster for the row, one to four CTAs, more rows than CTAs


def _case(B, V, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, V, generator=g) * scale).to(dtype).cuda()
    return x, torch.randint(V - 50, V, (B,), generator=g).cuda(), g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", SHAPES)
@pytest.mark.parametrize("mask", [-1e4, -5e4, -1e9, -1e10, -1e15, -1e20, -1e28, -1e35])
def test_masks(cuda_device, mask, B, V, dtype):
    if mask < float(torch.finfo(dtype).min):
        pytest.skip("below the type's lowest value")
    for T in (0.3, 1.0, 7.0, 1e-4):
        x, t, _ = _case(B, V, dtype, V)
        x[:, : V - 100] = mask                        # most threads see masked columns only
        temp = torch.full((B,), T, device="cuda")
        _check(x, t, temp, top=5)
        _check(x.flip(1), V - 1 - t, temp)
        g, h = torch.full((B,), 3.0, device="cuda"), torch.full((B,), 0.5, device="cuda")
        if T >= 0.3:
            d = _grad_case(x, t, temp, g, h, dtype)
            assert d.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", SHAPES)
def test_masks_of_many_sizes_in_one_row(cuda_device, B, V, dtype):
    x, t, g = _case(B, V, dtype, 1)
    low = float(torch.finfo(dtype).min)
    sizes = torch.tensor([max(v, low) for v in (-1e4, -3e4, -1e9, -1e10, -1e15, -1e20, -1e28, -1e35, low, -math.inf)])
    kinds = sizes[torch.randint(0, len(sizes), (B, V), generator=g)].to(dtype).cuda()
    kinds[:, -100:] = x[:, -100:]
    _check(kinds, t, None, top=5)
    _check(kinds, t, torch.full((B,), 0.01, device="cuda"))


@pytest.mark.parametrize("B,V", SHAPES)
@pytest.mark.parametrize("dtype,center,T", [
    (torch.float32, 3e9, 1.0), (torch.float32, -3e9, 1.0), (torch.float32, 3000.0, 1e-6), (torch.float32, 1e20, 1e10),
    (torch.float32, -1e30, 1e20), (torch.float16, 4e4, 1e-5), (torch.float16, -4e4, 1e-5), (torch.float16, -4e4, 0.02),
    (torch.float16, -6.2e4, 1.0), (torch.bfloat16, 1e12, 1.0), (torch.bfloat16, -1e12, 1e3), (torch.bfloat16, 100.0, 1e-7)])
def test_rows_far_from_zero(cuda_device, dtype, center, T, B, V):
    x, t, g = _case(B, V, torch.float32, 2)
    spacing = abs(center) * {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[dtype]
    y = (center + x * max(T, spacing)).to(dtype)
    _check(y, t, torch.full((B,), T, device="cuda"), top=4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", SHAPES)
@pytest.mark.parametrize("at", [2.0 ** 20, 2.0 ** 23 * 0.99, 2.0 ** 23 * 1.01, 2.0 ** 23.58, 2.0 ** 23.59, 2.0 ** 24 * 0.99,
                                2.0 ** 24 * 1.01, 2.0 ** 26])
def test_either_side_of_the_limits(cuda_device, at, B, V, dtype):
    """Rows whose logits are `at` halvings of the probability away from 0, above and below, with columns
    up to twice as far below them."""
    T = 1e-3 if dtype == torch.float16 else 0.5
    center = at * math.log(2.0) * T                      # f16: up to 46517
    for sign in (1.0, -1.0):
        x, t, g = _case(B, V, torch.float32, 3)
        y = center * sign + x * max(T, center * torch.finfo(dtype).eps)
        step = torch.randint(0, 9, (B, V), generator=g).cuda() * center / 8
        keep = torch.rand(B, V, generator=g).cuda() < 0.5
        keep[:, -100:] = True
        y = torch.where(keep, y, y - step).clamp(min=float(torch.finfo(dtype).min)).to(dtype)
        _check(y, t, torch.full((B,), T, device="cuda"), top=3)
