"""The adapters of the LM head where they are hard on the 16-bit operands: components of the inner
product of very unequal size, in every rank's layout."""
import pytest
import torch

from flashgen_b200.sampling.lm_head import AdapterHead

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _unequal(B, dtype, rank, spread, seed=0):
    """A head without shared weights whose component i of U is 2^-s_i times the first, s_i up to `spread`
    (32 columns of hidden each), and whose vocabulary row v takes component v % rank alone, at a size that
    makes up for it."""
    g = torch.Generator().manual_seed(seed + B + rank)
    n, V = 32, 4 * rank + 3
    size = [spread * i // max(1, rank - 1) for i in range(rank)]       # halvings of component i
    x = torch.randn(B, rank * n, generator=g)
    x = torch.where(x.abs() < 0.1, torch.full_like(x, 0.1), x)
    down = torch.zeros(rank, rank * n)
    up = torch.zeros(V, rank)
    for i, s in enumerate(size):
        # 2^6 (s = 0) to 2^-30, shared between hidden and down; up to 2^14 in up
        part = torch.randn(n, generator=g)
        x[:, i * n:(i + 1) * n] *= 2.0 ** (3 - s // 2)
        down[i, i * n:(i + 1) * n] = torch.where(part.abs() < 0.1, torch.full_like(part, 0.1), part) * 2.0 ** (3 - (s - s // 2))
        up[i::rank, i] = (0.5 + torch.rand(len(up[i::rank]), generator=g)) * 2.0 ** min(s - 8, 14)
    return x.to(dtype).cuda(), down.to(dtype).cuda(), up.to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [1, 40, 70, 300])
@pytest.mark.parametrize("rank,spread", [(2, 4), (2, 20), (2, 30), (8, 24), (8, 32), (16, 32), (24, 30), (33, 32), (65, 32),
                                         (100, 24), (128, 32)])
def test_components_of_unequal_size(cuda_device, dtype, B, rank, spread):
    """Every result is one component times one element of up, so the component's own precision shows: its
    sum of 32 products errs by at most 32 roundings of 2^-24 of the products' magnitudes, its parts keep
    2^-23 of it, the product and the scaling back round three times more. The other components meet zeros."""
    x, down, up = _unequal(B, dtype, rank, spread)
    V, dim = up.shape[0], x.shape[1]
    head = AdapterHead(torch.zeros(V, dim, dtype=dtype, device="cuda"), slots=2, rank=rank)
    head.load(1, down, up)
    ids = torch.ones(B, dtype=torch.int32, device="cuda")
    want = x.double() @ down.double().T @ up.double().T
    bound = 40 * 2.0 ** -24 * (x.double().abs() @ down.double().abs().T @ up.double().abs().T)
    got = head.logits(x, ids, out_dtype=torch.float32).double()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound.clamp_min(1e-300)).max()
    unit, tiny = (2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -8, 0.0)
    got = head.logits(x, ids).double()
    fits = want.abs() < 65504 if dtype == torch.float16 else torch.ones_like(want, dtype=torch.bool)
    assert ((got - want).abs() <= bound + want.abs() * unit + tiny)[fits].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [3, 70])
@pytest.mark.parametrize("power", [-40, -100, 40, 90])
def test_components_of_any_magnitude(cuda_device, dtype, B, power):
    """The scale takes U far from 1 as a whole: the sums keep their relative precision."""
    if dtype == torch.float16 and power == -100:
        power = -60
    x, down, up = _unequal(B, dtype, 8, 12)
    head = AdapterHead(torch.zeros(up.shape[0], x.shape[1], dtype=dtype, device="cuda"), slots=1, rank=8)
    head.load(0, down, up, scale=2.0 ** power)
    ids = torch.zeros(B, dtype=torch.int32, device="cuda")
    want = x.double() @ down.double().T @ up.double().T * 2.0 ** power
    bound = 40 * 2.0 ** -24 * (x.double().abs() @ down.double().abs().T @ up.double().abs().T) * 2.0 ** power
    got = head.logits(x, ids, out_dtype=torch.float32).double()
    assert ((got - want).abs() <= bound).all()
