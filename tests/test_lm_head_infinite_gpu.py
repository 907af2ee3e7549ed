"""Infinite elements of an adapter: a row's own give what the definition gives, infinity or NaN, and
everything finite stays exact."""
import math

import pytest
import torch

from tests.test_lm_head_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu


def _check(c):
    """Integer inputs (see Case): equal to the definition in 64 bits, infinities and NaN in the same places."""
    x = c.hidden.double()
    want = x @ c.weight.double().T
    for s in range(len(c.down)):
        rows = torch.nonzero(c.adapters == s)[:, 0]
        u = c.scale[s] * (x[rows] @ c.down[s].double().T)
        # a sum of products with infinities, one product at a time
        for i in range(u.shape[1]):
            want[rows] += u[:, i:i + 1] * c.up[s][:, i].double()[None, :]
    for out in (torch.float32, c.hidden.dtype):
        got = c.head.logits(c.hidden, c.adapters, out_dtype=out)
        torch.testing.assert_close(got.double(), want.float().to(out).double(), rtol=0, atol=0, equal_nan=True)
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 128])
@pytest.mark.parametrize("B", [1, 7, 40, 70, 300])
def test_infinite_up(cuda_device, B, rank, dtype):
    c = Case(B, 72, 300, rank, 3, dtype, bare=B > 1)
    inf = math.inf
    c.up[0][3, 2] = inf
    c.up[0][5, 0] = -inf
    c.up[0][40, 1] = inf
    c.up[0][40, 5] = inf                          # two: infinite or NaN by the components' signs
    c.up[1][299, 7] = inf
    c.up[1][129, :] = -inf
    c.up[2][0, 0] = float("nan")
    for s in range(3):
        c.head.load(s, c.down[s], c.up[s], c.scale[s])
    want = _check(c)
    if B >= 40:
        assert want.isinf().any() and want.isnan().any() and want.isfinite().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [5, 70])
def test_infinite_components(cuda_device, B, dtype):
    """An infinite component of U: infinite where up is not 0, NaN where it is; and beside a large finite one."""
    c = Case(B, 72, 300, 16, 2, dtype, bare=False)
    c.hidden.abs_().add_(1)                       # no zeros: the sums with infinities are infinite
    c.down[0].abs_().add_(1)
    c.down[1].abs_().add_(1)
    c.down[0][4, 10] = math.inf
    c.down[1][2, 0] = -math.inf
    c.up[1].abs_().add_(1)
    for s in range(2):
        c.head.load(s, c.down[s], c.up[s], c.scale[s])
    want = _check(c)
    assert want.isinf().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_components_meet_infinity(cuda_device, dtype):
    """A component far below the row's largest times an infinite element of up."""
    c = Case(9, 72, 300, 8, 1, dtype, bare=False)
    c.down[0].zero_()
    c.down[0][0, 0] = 1.0
    c.down[0][1, 1] = 2.0 ** -12
    c.hidden.fill_(0)
    c.hidden[:, 0] = 64
    c.hidden[:, 1] = -(2.0 ** -12)                # a component of -2^-24 beside one of 2^6
    c.up[0][:, 0] = 1
    c.up[0][7, 1] = math.inf
    c.head.load(0, c.down[0], c.up[0], 1.0)
    for out in (torch.float32, dtype):
        got = c.head.logits(c.hidden, c.adapters, out_dtype=out)
        assert (got[:, 7] == -math.inf).all()
        assert got[:, :7].isfinite().all() and got[:, 8:].isfinite().all()
