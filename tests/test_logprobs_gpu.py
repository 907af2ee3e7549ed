"""Token log probabilities, entropies, ranks and alternatives, and their
gradient, against the definitions in 64 bits (tests/logprob_reference.py)."""
import ctypes

import numpy as np
import pytest
import torch

from flashgen_b200 import _lib
from flashgen_b200.sampling.logprobs import logprobs_and_entropy, token_logprobs, token_logprobs_grad
from tests import logprob_reference as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _name(dtype):
    return str(dtype).split(".")[1]


def _check(logits, tokens, temperature=None, top=0):
    """logits on the GPU (any strides); compares every output."""
    B, V = logits.shape
    T = np.ones(B) if temperature is None else temperature.double().cpu().numpy()
    tok = np.full(B, -1) if tokens is None else tokens.cpu().numpy()
    r = token_logprobs(logits, tokens, temperature=temperature, top=top)
    ref = R.forward(logits.double().cpu().numpy(), tok, T, top)
    got = {k: getattr(r, k).double().cpu().numpy() for k in ("logprobs", "entropy", "max", "logsum")}
    np.testing.assert_array_equal(got["max"], ref["max"])
    np.testing.assert_array_equal(r.rank.cpu().numpy(), ref["rank"])
    ym = ref["ymax"]
    _close(got["logsum"], ref["logsum"], R.logprob_bound(V, ym, 0.0))
    _close(got["logprobs"], ref["logprobs"], R.logprob_bound(V, ym, ref["logprobs"]))
    _close(got["entropy"], ref["entropy"], R.entropy_bound(V, ym))
    if top:
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ref["top_ids"])
        _close(r.top_logprobs.double().cpu().numpy(), ref["top_logprobs"],
               R.logprob_bound(V, ym[:, None], ref["top_logprobs"]))
    else:
        assert r.top_ids is None and r.top_logprobs is None
    empty = ref["max"] == -np.inf
    np.testing.assert_array_equal(r.status.cpu().numpy(), np.where(empty, _lib.FG_ROW_ALL_MASKED, 0))
    return r


def _close(got, want, bound):
    bound = np.broadcast_to(bound, np.shape(want))
    with np.errstate(over="ignore"):
        want = np.where(np.isinf(np.float32(want)), np.float32(want), want)   # beyond fp32: infinite
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])
    err = np.abs(got - np.where(inf, got, want))
    ok = inf | (err <= bound)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5], bound[~ok][:5])


def _random(B, V, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, V, generator=g) * scale).to(dtype).cuda()
    t = torch.randint(0, V, (B,), generator=g).cuda()
    T = (0.5 + torch.rand(B, generator=g)).cuda()
    return x, t, T


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 31, 33, 257, 1000, 4097, 12289, 50257])
def test_forward_sizes(cuda_device, V, dtype):
    x, t, T = _random(5, V, dtype, V)
    t[1] = -1
    _check(x, t, T, top=min(20, V + 2, 32))
    _check(x, t, None, top=0)


@pytest.mark.parametrize("B", [1, 2, 17, 64, 149, 300])
def test_forward_batches(cuda_device, B):
    x, t, T = _random(B, 9001, torch.bfloat16, B)
    _check(x, t, T, top=5)


@pytest.mark.parametrize("top", [0, 1, 2, 5, 20, 31, 32])
def test_forward_top(cuda_device, top):
    for dtype, V in ((torch.float32, 128256), (torch.bfloat16, 32000)):
        x, t, T = _random(3, V, dtype, top)
        _check(x, t, T, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 2), (3, 8), (5, 3), (8, 8)])
def test_forward_unaligned(cuda_device, dtype, offset, pad):
    g = torch.Generator().manual_seed(offset)
    B, V = 6, 9001
    big = (torch.randn(B, V + offset + pad, generator=g) * 3).to(dtype).cuda()
    t = torch.randint(0, V, (B,), generator=g).cuda()
    _check(big[:, offset:offset + V], t, None, top=9)
    _check(big[::2, offset:offset + V], t[::2], None, top=9)     # every second row
    _check(big.t().contiguous().t()[:, offset:offset + V], t, None, top=3)   # columns not dense: copied


@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_large_logits(cuda_device, dtype):
    # an offset common to the row changes nothing; differences of hundreds underflow to exact zeros
    x, t, T = _random(4, 5003, dtype, 1, scale=3.0)
    _check((x.float() + 1000).to(dtype), t, T, top=4)
    _check((x.float() - 1000).to(dtype), t, T, top=4)
    _check((x.float() * 300).to(dtype), t, T, top=4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1e-30, 1e-6, 1e-3, 0.02, 50.0, 1e4, 1e30])
def test_forward_temperatures(cuda_device, dtype, T):
    x, t, _ = _random(4, 4099, dtype, 2)
    x[1, 5:] = -float("inf")
    x[2, ::2] = torch.finfo(dtype).min
    t[1], t[2] = 2, 7
    _check(x, t, torch.full((4,), T, device="cuda"), top=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [6, 4099, 50257])
def test_forward_masks(cuda_device, dtype, V):
    x, t, T = _random(10, V, dtype, V)
    low, ninf = torch.finfo(dtype).min, -float("inf")
    x[0] = ninf                                   # empty
    x[1, 1:] = ninf; t[1] = 0                     # one id left
    x[2, : V - 1] = ninf; t[2] = 0                # one id left, the token masked
    x[3] = low                                    # the type's lowest value everywhere: uniform
    x[4, 2:] = low; t[4] = 1
    x[5, 3:] = low; t[5] = V - 1                  # the token masked with it
    x[6, ::2] = ninf; x[6, 1::2] = low; t[6] = 1  # lowest among -inf
    x[7, : V // 2] = ninf
    x[8] = torch.finfo(dtype).max                 # the type's largest value everywhere
    x[9] = ninf; t[9] = -1                        # empty, no token
    for top in (0, 2, 5):
        _check(x, t, None, top=top)
        _check(x, t, T, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_ties(cuda_device, dtype):
    V = 8191
    x = torch.zeros(6, V, dtype=dtype, device="cuda")     # every logit alike: ids in order
    x[1] = -0.0
    x[1, ::3] = 0.0                                       # zeros of both signs are equal
    x[2] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(0)).to(dtype)
    x[3, 4000:4100] = 2
    x[4, -1] = 1                                          # the last column, in the ragged end
    x[5] = torch.arange(V).to(dtype) / 64                 # ascending, with ties in 16 bits
    t = torch.tensor([8190, 1, 77, 4050, 8190, 100], device="cuda")
    for top in (1, 20, 32):
        _check(x, t, None, top=top)
        _check(x.flip(1), t, None, top=top)


def test_forward_special_rows(cuda_device):
    x, t, T = _random(8, 1237, torch.float32, 3)
    x[0, 100] = float("nan")
    x[1, 1236] = float("inf")
    x[2, 0] = float("nan"); x[2, 1] = float("inf")
    T[3], T[4], T[5] = 0.0, float("nan"), float("inf")
    t[6] = 1237
    r = token_logprobs(x, t, temperature=T, top=3)
    st = r.status.cpu().tolist()
    assert st == [_lib.FG_ROW_NAN, _lib.FG_ROW_POS_INF, _lib.FG_ROW_NAN] + [_lib.FG_ROW_BAD_PARAM] * 4 + [0]
    for k in ("logprobs", "entropy", "logsum"):
        v = getattr(r, k)
        assert v[:7].isnan().all() and v[7].isfinite(), k
    assert (r.rank[:7] == -1).all() and (r.top_ids[:7] == -1).all() and r.top_logprobs[:7].isnan().all()
    _check(x[7:], t[7:], T[7:], top=3)
    with pytest.raises(RuntimeError, match="row 0"):
        token_logprobs(x, t, temperature=T, check_errors=True)


def test_forward_repeats_and_streams(cuda_device):
    x, t, T = _random(40, 50257, torch.bfloat16, 4)
    a = token_logprobs(x, t, temperature=T, top=20)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = token_logprobs(x, t, temperature=T, top=20)
    torch.cuda.synchronize()
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def test_forward_row_offsets_pass_32_bits(cuda_device):
    # the last row starts more than 2^32 bytes into the buffer
    V, stride, B = 1025, 1 << 22, 520
    buf = torch.empty(B * stride, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((B, V), (stride, 1))
    x.copy_(_random(B, V, torch.bfloat16, 5)[0])
    t = torch.arange(B, device="cuda")
    _check(x, t, None, top=2)
    g = torch.ones(B, device="cuda")
    r = token_logprobs(x, t)
    a = token_logprobs_grad(x, t, r.max, r.logsum, g)
    assert torch.equal(a, token_logprobs_grad(x.contiguous(), t, r.max, r.logsum, g))
    token_logprobs_grad(x, t, r.max, r.logsum, g, out=x)
    assert torch.equal(a, x)


def _grad_case(x, t, T, g, h, dtype):
    Tn = np.ones(len(x)) if T is None else T.double().cpu().numpy()
    xn = x.double().cpu().numpy()
    r = token_logprobs(x, t, temperature=T)
    d = token_logprobs_grad(x, t, r.max, r.logsum, g, entropy=r.entropy, grad_entropy=h, temperature=T)
    assert d.dtype == dtype and d.shape == x.shape
    tok = t.cpu().numpy()
    ref = R.forward(xn, tok, Tn, 0)
    gn = np.zeros(len(x)) if g is None else g.double().cpu().numpy()
    want, size = R.gradient(xn, tok, Tn, gn, None if h is None else h.double().cpu().numpy())
    # the saved statistics come from the forward kernel: its bounds enter as relative errors of p
    extra = (R.logprob_bound(x.shape[1], ref["ymax"], 0.0) + R.entropy_bound(x.shape[1], ref["ymax"]))[:, None]
    bound = R.gradient_bound(want, size, x.shape[1], ref["ymax"], _name(dtype)) + extra * size
    _close(d.double().cpu().numpy(), want, bound)
    return d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 33, 257, 4097, 50257])
def test_gradient_sizes(cuda_device, V, dtype):
    B = 7
    x, t, T = _random(B, V, dtype, V)
    t[2] = -1
    gen = torch.Generator().manual_seed(V)
    g = (torch.randn(B, generator=gen) * 64).cuda()
    h = torch.randn(B, generator=gen).cuda()
    g[4] = 0; h[4] = 0
    d = _grad_case(x, t, T, g, h, dtype)
    assert (d[4] == 0).all()
    _grad_case(x, t, None, g, None, dtype)
    _grad_case(x, t, T, None, h, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,pad,opad", [(0, 1, 0), (1, 2, 1), (3, 8, 5), (5, 3, 3), (8, 8, 0)])
def test_gradient_unaligned(cuda_device, dtype, offset, pad, opad):
    gen = torch.Generator().manual_seed(offset)
    B, V = 6, 4099
    big = (torch.randn(B, V + offset + pad, generator=gen) * 3).to(dtype).cuda()
    x = big[:, offset:offset + V]
    t = torch.randint(0, V, (B,), generator=gen).cuda()
    g, h = torch.randn(B, generator=gen).cuda() * 32, torch.randn(B, generator=gen).cuda()
    d = _grad_case(x, t, None, g, h, dtype)
    r = token_logprobs(x, t)
    kw = dict(entropy=r.entropy, grad_entropy=h)
    room = torch.full((B, V + 2 * opad + 1), 7.0, dtype=dtype, device="cuda")
    out = room[:, opad:opad + V]
    token_logprobs_grad(x, t, r.max, r.logsum, g, out=out, **kw)
    assert torch.equal(out, d)
    assert (room[:, :opad] == 7).all() and (room[:, opad + V:] == 7).all()      # nothing outside the rows
    keep = big.clone()
    token_logprobs_grad(x, t, r.max, r.logsum, g, out=x, **kw)                  # over the logits
    assert torch.equal(x, d)
    assert torch.equal(big[:, :offset], keep[:, :offset]) and torch.equal(big[:, offset + V:], keep[:, offset + V:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_masks(cuda_device, dtype):
    V = 4099
    x, t, T = _random(9, V, dtype, 6)
    low, ninf = torch.finfo(dtype).min, -float("inf")
    x[0] = ninf
    x[1, 1:] = ninf; t[1] = 0
    x[2, : V - 1] = ninf; t[2] = 0
    x[3] = low
    x[4, 2:] = low; t[4] = 1
    x[5, 3:] = low; t[5] = V - 1
    x[6, ::2] = ninf; x[6, 1::2] = low; t[6] = 1
    x[7] = torch.finfo(dtype).max
    g, h = torch.full((9,), 3.0, device="cuda"), torch.full((9,), 0.5, device="cuda")
    for temp in (None, T):
        d = _grad_case(x, t, temp, g, h, dtype)
        assert (d[0] == 0).all() and (d[6, ::2] == 0).all()


def test_gradient_special_rows(cuda_device):
    x, t, T = _random(6, 777, torch.float32, 7)
    x[0, 3] = float("nan"); x[1, 4] = float("inf"); T[2] = -1.0; t[3] = 777
    x[4, 5] = float("nan")
    g = torch.ones(6, device="cuda"); g[4] = 0
    r = token_logprobs(x, t, temperature=T)
    d = token_logprobs_grad(x, t, r.max, r.logsum, g, temperature=T)
    assert d[:4].isnan().all()
    assert (d[4] == 0).all()          # nothing flows into the row: exactly zero whatever it holds
    assert d[5].isfinite().all()


def test_autograd_matches_differences(cuda_device):
    """The gradient against central differences of the 64-bit definition."""
    B, V = 3, 13
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(B, V, generator=gen)
    t = torch.tensor([4, -1, 12])
    T = torch.tensor([0.7, 1.0, 1.5])
    g, h = torch.randn(B, generator=gen), torch.randn(B, generator=gen)
    xg = x.cuda().requires_grad_()
    lp, ent = logprobs_and_entropy(xg, t.cuda(), T.cuda())
    ((g.cuda() * lp).sum() + (h.cuda() * ent).sum()).backward()

    def value(z):
        f = R.forward(z, t.numpy(), T.double().numpy(), 0)
        return (g.double().numpy() * f["logprobs"]).sum() + (h.double().numpy() * f["entropy"]).sum()

    xn, eps = x.double().numpy(), 1e-5
    num = np.zeros((B, V))
    for r in range(B):
        for j in range(V):
            hi, lo = xn.copy(), xn.copy()
            hi[r, j] += eps
            lo[r, j] -= eps
            num[r, j] = (value(hi) - value(lo)) / (2 * eps)
    # differences: eps^2 times third derivatives (of order 10) plus 1e-16 / eps; fp32: 1e-6 of order-1 terms
    np.testing.assert_allclose(xg.grad.cpu().numpy(), num, atol=1e-5)


def test_autograd_broadcast_and_unused(cuda_device):
    x, t, _ = _random(5, 101, torch.float32, 9)
    a = x.clone().requires_grad_()
    lp, _ = logprobs_and_entropy(a, t)
    lp.sum().backward()                                     # an expanded upstream gradient
    b = x.clone().requires_grad_()
    torch.log_softmax(b, 1).gather(1, t[:, None]).sum().backward()
    # both sides in fp32 on terms below 1
    torch.testing.assert_close(a.grad, b.grad, atol=2e-6, rtol=0)
    row = x[:1].clone().requires_grad_()                    # one row shared by the batch: gradients add up
    lp, ent = logprobs_and_entropy(row.expand(5, 101), t)
    (lp.sum() + ent.sum()).backward()
    ref = x[:1].double().clone().requires_grad_()
    z = torch.log_softmax(ref.expand(5, 101), 1)
    (z.gather(1, t[:, None]).sum() - (z.exp() * z).sum()).backward()
    torch.testing.assert_close(row.grad.double(), ref.grad, atol=2e-5, rtol=0)
    c = x.clone().requires_grad_()
    lp, ent = logprobs_and_entropy(c, t)
    ent.sum().backward()                                    # only the entropy is used
    assert c.grad.isfinite().all()


def test_refusals(cuda_device):
    x, t, T = _random(4, 100, torch.float32, 10)
    r = token_logprobs(x, t)
    with pytest.raises(ValueError):
        token_logprobs(x[0], t)
    with pytest.raises(ValueError):
        token_logprobs(x, t[:3])
    with pytest.raises(ValueError):
        token_logprobs(x, t.cpu())
    with pytest.raises(ValueError):
        token_logprobs(x, t, top=33)
    with pytest.raises(ValueError):
        token_logprobs(x, t, top=-1)
    with pytest.raises(TypeError):
        token_logprobs(x, t.float())
    with pytest.raises(TypeError):
        token_logprobs(x, t, temperature=t)
    with pytest.raises(RuntimeError):
        token_logprobs(x.cpu(), t.cpu())
    with pytest.raises(ValueError):
        token_logprobs_grad(x, t, r.max, r.logsum, r.logprobs, grad_entropy=r.entropy)
    with pytest.raises(ValueError):
        token_logprobs_grad(x, t, r.max, r.logsum, r.logprobs, out=x.half())
    with pytest.raises(ValueError):
        token_logprobs_grad(x, t, r.max, r.logsum[:2], r.logprobs)
    empty = token_logprobs(x[:0], t[:0], top=3)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_c_abi_optional_outputs(cuda_device):
    """Every output may be absent."""
    lib = _lib.load()
    x, t, _ = _random(3, 5000, torch.float16, 11)
    full = token_logprobs(x, t, top=4)
    lp = torch.empty(3, device="cuda")
    ids = torch.empty(3, 4, dtype=torch.int64, device="cuda")
    a = _lib.FgLogprobArgs()
    a.logits, a.dtype, a.batch, a.vocab, a.row_stride = x.data_ptr(), _lib.FG_DTYPE_F16, 3, 5000, 5000
    st = torch.cuda.current_stream().cuda_stream
    assert lib.fg_token_logprobs(ctypes.byref(a), st) == _lib.FG_OK      # nothing to write
    a.tokens, a.out_logprobs = t.data_ptr(), lp.data_ptr()
    a.top = 4                                                            # no place for them: not computed
    assert lib.fg_token_logprobs(ctypes.byref(a), st) == _lib.FG_OK
    a.out_top_ids = ids.data_ptr()
    assert lib.fg_token_logprobs(ctypes.byref(a), st) == _lib.FG_OK
    torch.cuda.synchronize()
    assert torch.equal(lp, full.logprobs) and torch.equal(ids, full.top_ids)
