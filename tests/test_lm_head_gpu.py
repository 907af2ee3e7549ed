"""The LM head with per-row low-rank adapters against its definition in 64
bits. Most inputs are small integers (and scales powers of two), so that every
product and every partial sum is exact in fp32 and the result is one rounding
of the exact one: those tests ask for equality."""
import ctypes

import pytest
import torch

from flashgen_b200 import _lib
from flashgen_b200.sampling.lm_head import AdapterHead

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _ints(shape, lo, hi, dtype, gen):
    return torch.randint(lo, hi + 1, shape, generator=gen).to(dtype).cuda()


class Case:
    """Integer inputs: |sums| stay below 2^20."""

    def __init__(self, B, dim, V, rank, slots, dtype, seed=0, bare=True):
        g = torch.Generator().manual_seed(seed + 1000 * B + dim)
        self.hidden = _ints((B, dim), -2, 2, dtype, g)
        self.weight = _ints((V, dim), -3, 3, dtype, g)
        self.head = AdapterHead(self.weight, slots=slots, rank=rank)
        self.down = [_ints((rank, dim), -1, 1, dtype, g) for _ in range(slots)]
        self.up = [_ints((V, rank), -2, 2, dtype, g) for _ in range(slots)]
        self.scale = [0.5 * (1 + s % 3) if s % 3 < 2 else 2.0 for s in range(slots)]
        for s in range(slots):
            self.head.load(s, self.down[s], self.up[s], self.scale[s])
        self.adapters = torch.randint(-1 if bare else 0, max(1, slots), (B,), generator=g).to(torch.int32).cuda()
        if slots == 0:
            self.adapters.fill_(-1)

    def exact(self, adapters=True):
        x = self.hidden.double()
        out = x @ self.weight.double().T
        if adapters:
            for s in range(len(self.down)):
                rows = torch.nonzero(self.adapters == s)[:, 0]
                if rows.numel():
                    out[rows] += self.scale[s] * (x[rows] @ self.down[s].double().T) @ self.up[s].double().T
        return out

    def check(self):
        want = self.exact()
        got = self.head.logits(self.hidden, self.adapters, out_dtype=torch.float32)
        assert got.dtype == torch.float32
        assert torch.equal(got.double(), want), (got.double() - want).abs().max()
        got = self.head.logits(self.hidden, self.adapters)
        assert torch.equal(got, want.float().to(self.hidden.dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256,
                               257, 300, 511, 513, 700])
def test_batches(cuda_device, B, dtype):
    Case(B, 200, 391, 16, 4, dtype).check()


@pytest.mark.parametrize("dim", [1, 2, 7, 8, 15, 16, 17, 63, 64, 65, 127, 128, 129, 192, 448, 1000, 1001, 2056])
def test_dims(cuda_device, dim):
    for B in (1, 5, 70):
        Case(B, dim, 260, 8, 3, torch.bfloat16).check()


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 127, 128, 129, 255, 256, 257, 1000, 5003, 40000])
def test_vocabularies(cuda_device, V):
    for B in (1, 19, 130):
        Case(B, 136, V, 16, 3, torch.float16).check()


@pytest.mark.parametrize("rank", [1, 4, 8, 15, 16, 17, 32, 40, 64, 65, 100, 128])
def test_ranks(cuda_device, rank):
    for B in (1, 40, 300):
        Case(B, 72, 300, rank, 3, torch.bfloat16).check()


@pytest.mark.parametrize("slots", [0, 1, 2, 16, 40, 300])
def test_slots(cuda_device, slots):
    # as many adapters as rows, one adapter for all, more slots than rows
    Case(64, 80, 300, 16, slots, torch.bfloat16).check()
    Case(300, 80, 300, 16, slots, torch.float16, bare=False).check()


def test_one_adapter_in_many_orders(cuda_device):
    c = Case(290, 96, 500, 16, 8, torch.bfloat16)
    for a in (torch.zeros(290), torch.arange(290) % 8, (torch.arange(290) // 40).clamp_max(7),
              torch.full((290,), -1.0), torch.where(torch.arange(290) == 137, 5, -1)):
        c.adapters = a.to(torch.int32).cuda()
        c.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [1, 37, 300])
@pytest.mark.parametrize("dim", [256, 1000, 4096])
def test_real_values(cuda_device, dtype, B, dim):
    """fp32 sums of 16-bit products: a sum of n terms taken 16 at a time errs by at most
    (n / 16 + 16) 2^-23 of the sum of the terms' magnitudes, also where the adder truncates."""
    g = torch.Generator().manual_seed(B + dim)
    V, r = 3001, 24

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()

    weight, hidden = normal(V, dim, scale=dim ** -0.5), normal(B, dim)
    head = AdapterHead(weight, slots=2, rank=r)
    down, up = [normal(r, dim, scale=dim ** -0.5) for _ in range(2)], [normal(V, r, scale=0.1) for _ in range(2)]
    for s in range(2):
        head.load(s, down[s], up[s], 1.5)
    ad = (torch.arange(B) % 3 - 1).to(torch.int32).cuda()
    x = hidden.double()
    want, size = x @ weight.double().T, x.abs() @ weight.double().abs().T
    steps = dim / 16 + 16
    bound = steps * 2.0 ** -23 * size
    for s in range(2):
        rows = torch.nonzero(ad == s)[:, 0]
        u = 1.5 * x[rows] @ down[s].double().T
        want[rows] += u @ up[s].double().T
        usize = 1.5 * x[rows].abs() @ down[s].double().abs().T
        bound[rows] += (steps + r + 4) * 2.0 ** -23 * (usize @ up[s].double().abs().T)
    got = head.logits(hidden, ad, out_dtype=torch.float32)
    assert ((got.double() - want).abs() <= bound + want.abs() * 2.0 ** -23).all()
    got16 = head.logits(hidden, ad)
    unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    assert ((got16.double() - want).abs() <= bound + want.abs() * unit + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(cuda_device, dtype):
    for B in (3, 150):
        c = Case(B, 130, 301, 16, 3, dtype)
        want = c.exact()
        for off, pad in ((0, 6), (1, 0), (3, 2), (8, 6)):
            room = torch.zeros(B, off + 130 + pad, dtype=dtype, device="cuda")
            room[:, off:off + 130] = c.hidden
            got = c.head.logits(room[:, off:off + 130], c.adapters, out_dtype=torch.float32)
            assert torch.equal(got.double(), want)
        got = c.head.logits(c.hidden.t().contiguous().t(), c.adapters, out_dtype=torch.float32)
        assert torch.equal(got.double(), want)
        room = torch.full((B, 301 + 9), 7.0, dtype=dtype, device="cuda")     # an output inside a larger buffer
        c.head.logits(c.hidden, c.adapters, out=room[:, 5:306])
        assert torch.equal(room[:, 5:306], want.float().to(dtype))
        assert (room[:, :5] == 7).all() and (room[:, 306:] == 7).all()
        # weights whose rows are not 16-byte aligned are laid out once
        wide = torch.zeros(301, 133, dtype=dtype, device="cuda")
        wide[:, 2:132] = c.weight
        head = AdapterHead(wide[:, 2:132])
        got = head.logits(c.hidden, out_dtype=torch.float32)
        assert torch.equal(got.double(), c.exact(adapters=False))


def test_adapters_are_apart(cuda_device):
    """NaN and inf in one request's adapter or hidden row reach no other row."""
    for B in (4, 64, 300):
        c = Case(B, 100, 300, 16, 4, torch.bfloat16)
        c.adapters = (torch.arange(B) % 4).to(torch.int32).cuda()
        want = c.exact()
        c.up[1][:] = float("nan"); c.up[2][:, 3] = float("inf")
        c.down[2][:] = 1
        for s in (1, 2):
            c.head.load(s, c.down[s], c.up[s], 1.0)
        hidden = c.hidden.clone()
        hidden[3] = float("nan")
        got = c.head.logits(hidden, c.adapters, out_dtype=torch.float32)
        rows = torch.nonzero((c.adapters != 1) & (c.adapters != 2))[:, 0]
        rows = rows[rows != 3]
        assert torch.equal(got[rows].double(), want[rows])
        assert got[1].isnan().all() and got[3].isnan().all()


def test_load_replaces_and_unload_empties(cuda_device):
    c = Case(20, 64, 200, 16, 2, torch.float16, bare=False)
    c.down[0], c.up[0] = c.down[0][:5], c.up[0][:, :5]          # a lower rank over a higher one
    c.scale[0] = 1.0
    c.head.load(0, c.down[0], c.up[0])
    c.check()
    c.head.unload(1)
    c.adapters = torch.where(c.adapters == 1, torch.full_like(c.adapters, -1), c.adapters)
    want = c.exact()
    back = torch.where(c.adapters < 0, torch.full_like(c.adapters, 1), c.adapters)   # still naming the empty slot
    assert torch.equal(c.head.logits(c.hidden, back, out_dtype=torch.float32).double(), want)


def test_bad_slots(cuda_device):
    c = Case(6, 64, 200, 16, 2, torch.float16, bare=False)
    c.adapters[2], c.adapters[4] = 2, 1 << 30
    plain = c.exact()
    got = c.head.logits(c.hidden, c.adapters, out_dtype=torch.float32)
    assert torch.equal(got.double(), plain)          # rows 2 and 4: the shared logits alone
    with pytest.raises(RuntimeError, match="row 2.*2 row"):
        c.head.logits(c.hidden, c.adapters, check_errors=True)
    c.adapters[2] = c.adapters[4] = -5
    c.head.logits(c.hidden, c.adapters, check_errors=True)


def test_streams_and_graphs(cuda_device):
    c = Case(33, 256, 1000, 16, 3, torch.bfloat16)
    want = c.exact()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.head.logits(c.hidden, c.adapters, out_dtype=torch.float32)
    s.synchronize()
    assert torch.equal(got.double(), want)
    out = torch.zeros(33, 1000, dtype=torch.float32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.head.logits(c.hidden, c.adapters, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.double(), want)
    c.hidden.neg_()                                   # the captured call reads its inputs anew
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.double(), -want)


def test_refusals(cuda_device):
    w = torch.zeros(100, 64, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        AdapterHead(w.float())
    with pytest.raises(RuntimeError):
        AdapterHead(w.cpu())
    with pytest.raises(ValueError):
        AdapterHead(w[0])
    with pytest.raises(ValueError):
        AdapterHead(w, slots=1, rank=129)
    head = AdapterHead(w, slots=2, rank=8)
    with pytest.raises(IndexError):
        head.load(2, w[:8], w[:, :8])
    with pytest.raises(ValueError):
        head.load(0, w[:9], w[:, :9])                 # rank above the bank's
    with pytest.raises(ValueError):
        head.load(0, w[:8, :63], w[:, :8])
    with pytest.raises(ValueError):
        head.logits(h[:, :63], ids)
    with pytest.raises(TypeError):
        head.logits(h.half(), ids)
    with pytest.raises(ValueError):
        head.logits(h, ids.long())
    with pytest.raises(ValueError):
        head.logits(h, ids[:3])
    with pytest.raises(TypeError):
        head.logits(h, ids, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        head.logits(h, ids, out=torch.zeros(4, 99, device="cuda"))
    assert head.logits(h[:0], ids[:0]).shape == (0, 100)
    lib = _lib.load()
    a = _lib.FgAdapterArgs()
    assert lib.fg_adapter_logits(ctypes.byref(a), None) == _lib.FG_EINVAL
