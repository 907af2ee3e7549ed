"""A wait of the linear block's kernel that runs out: what was not computed is NaN, nothing is left
unwritten, the call returns and the next one is as ever. The products of one accumulator are
computed and never reported (fg_linear_set_wait), so the wait for them ends at its limit of 5 ms."""
import pytest
import torch

from flashgen_b200 import _lib
from flashgen_b200.sampling import linear
from test_linear_gpu import BF16, F16, tensors

pytestmark = pytest.mark.gpu


@pytest.fixture
def withheld():
    lib = _lib.load()

    def set_(accumulator):
        torch.cuda.synchronize()
        assert lib.fg_linear_set_wait(5_000_000 if accumulator >= 0 else 0, accumulator) == _lib.FG_OK
    yield set_
    torch.cuda.synchronize()
    assert lib.fg_linear_set_wait(0, -1) == _lib.FG_OK


# one CTA a tile, sums split over a cluster (few tokens), pairs (many), one tile a CTA and
# several, sums in one piece and in several
@pytest.mark.parametrize("size,dtype,several", [
    ((1, 64, 100), BF16, False), ((1, 4096, 4096), BF16, False), ((1, 20000, 512), F16, False),
    ((64, 4096, 4096), F16, False), ((256, 4096, 4096), BF16, False), ((512, 4096, 4096), BF16, False),
    ((1024, 4096, 4096), F16, False), ((2048, 4096, 4096), BF16, True), ((8192, 512, 4096), F16, True),
    ((1000, 72, 40000), BF16, True), ((1024, 9000, 2048), F16, None)])
@pytest.mark.parametrize("accumulator", [0, 1])
def test_forward(cuda_device, withheld, size, dtype, several, accumulator):
    x, w, b, r, _ = tensors(*size, dtype, seed=31)
    act = linear._ACTIVATIONS["gelu"]
    want, _, _, z = linear._forward(x, w, b, r, act, True)
    z = z[:, :size[2]]
    withheld(accumulator)
    got, _, _, y = linear._forward(x, w, b, r, act, True)
    torch.cuda.synchronize()
    y = y[:, :size[2]]
    for g, a in ((got, want), (y, z)):
        lost = g.isnan()
        assert (lost | (g == a)).all()                  # the rest is right, nothing is unwritten
        if accumulator == 0:
            assert lost.all()
        elif several:
            assert lost.any() and not lost.all()        # the first tiles came through
        elif several is False and size[1] <= 4096:
            assert not lost.any()                       # one accumulation a CTA
    assert torch.equal(got.isnan(), y.isnan())
    withheld(-1)
    assert torch.equal(linear._forward(x, w, b, r, act, True)[0], want)


@pytest.mark.parametrize("size,dtype", [((40, 200, 300), F16), ((300, 77, 501), BF16), ((2048, 4096, 4096), BF16)])
def test_gradients(cuda_device, withheld, size, dtype):
    x, w, b, r, gy = tensors(*size, dtype, seed=32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    out = linear.fused_linear(*leaves, r, activation="silu")
    want = torch.autograd.grad(out, leaves, gy, retain_graph=True)
    withheld(0)
    got = torch.autograd.grad(out, leaves, gy, retain_graph=True)
    torch.cuda.synchronize()
    assert got[0].isnan().all() and got[1].isnan().all() and torch.equal(got[2], want[2])    # the bias's takes no product
    withheld(-1)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(out, leaves, gy), want))
