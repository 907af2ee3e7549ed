"""fp32 results of a long dim are summed in pieces: the tensor core truncates when it accumulates, and the
loss must not grow with dim."""
import pytest
import torch

from flashgen_b200.sampling.lm_head import AdapterHead

pytestmark = pytest.mark.gpu

PIECE = 512          # elements of a piece
STEP = 16            # products that the tensor core adds at a time


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B", [1, 40, 200])
def test_long_sums_of_one_sign(cuda_device, B, dtype):
    """All products positive, so every truncation goes the same way. Within a piece each of its steps, and
    each of the 16 products of one, may lose a unit of 2^-23 of what is there: (512 / 16 + 16) 2^-23 in all.
    The pieces are added with rounding, 2^-24 each. A sum in one piece loses 1500 2^-23, nineteen times this."""
    dim, V = 32768, 300
    g = torch.Generator().manual_seed(B)
    hidden = (0.5 + 0.5 * torch.rand(B, dim, generator=g)).to(dtype).cuda()
    weight = ((0.5 + 0.5 * torch.rand(V, dim, generator=g)) / 64).to(dtype).cuda()
    want = hidden.double() @ weight.double().T
    got = AdapterHead(weight).logits(hidden, out_dtype=torch.float32).double()
    bound = ((PIECE / STEP + STEP) * 2.0 ** -23 + dim / PIECE * 2.0 ** -24) * want
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / want).max() * 2 ** 23


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B", [1, 40, 100, 200, 300])
@pytest.mark.parametrize("dim", [4096, 4104, 32768, 65536])
def test_long_sums_of_one_sign_rounded(cuda_device, dim, B, dtype):
    """16-bit results: one rounding, and what pieces of 4096 may lose before it, (4096 / 16 + 16) 2^-23, with
    2^-24 for each piece added. In one piece 65536 products lose some 3000 2^-23, most of a float16 rounding."""
    V = 300
    g = torch.Generator().manual_seed(B)
    hidden = (0.5 + 0.5 * torch.rand(B, dim, generator=g)).to(dtype).cuda()
    weight = ((0.5 + 0.5 * torch.rand(V, dim, generator=g)) * (2.0 / dim) ** 0.5).to(dtype).cuda()
    want = hidden.double() @ weight.double().T
    head = AdapterHead(weight, slots=1, rank=8)
    got = head.logits(hidden).double()
    digits = 11 if dtype == torch.float16 else 8
    half_unit = 2.0 ** (torch.floor(torch.log2(want)) - digits)
    bound = half_unit + (272 * 2.0 ** -23 + dim / 4096 * 2.0 ** -24) * want
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / want).max() * 2 ** 23
    # and with an adapter that adds a column of hidden: one more rounding before the last
    down = torch.zeros(8, dim)
    down[0, 0] = 1
    head.load(0, down, torch.ones(V, 8))
    want = want + hidden[:, :1].double()
    got = head.logits(hidden, torch.zeros(B, dtype=torch.int32, device="cuda")).double()
    half_unit = 2.0 ** (torch.floor(torch.log2(want)) - digits)
    assert ((got - want).abs() <= half_unit + (273 * 2.0 ** -23 + dim / 4096 * 2.0 ** -24) * want).all()
