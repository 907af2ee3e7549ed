"""The fused linear block and its gradients against their definitions in 64 bits.

Tolerances, element by element, h being half a step of the type (eps / 2):
* a sum of products: the tensor core loses up to 0.05 n units of 2^-23 over n elements of a
  piece (at most p = 4096 of float16, 16384 of bfloat16), and a few more in the additions after
  it, of the sum of magnitudes S: e(S) = (0.05 min(n, p) + 4 + n / p) 2^-23 S;
* the activations' slopes are at most 1.13, and their own error a few units in 2^-22 of
  the larger of |act(z)| and |z| 2^-3 (e^x by a product and ex2, one division): 2^-20 of it;
* the result: h of itself, or half the least subnormal step;
* dz carries h of itself into the sums of the gradients: h S on top, in the worst case.
  The rounding errors of the summands are independent and at most h / sqrt(3) in the mean
  square, as is the result's own rounding: together 0.82 h of the result's norm. The
  gradients' norm of errors must be below h.
"""
import math

import pytest
import torch

from flashgen_b200 import HeadBlock, fused_linear

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
f = torch.nn.functional
# (gelu by the complementary error function: 1 + erf(z / sqrt 2) is 0 in 64 bits below z = -8.4, where
# the normal distribution is not: 1.8e-33 at -12)
ACTS = {"none": lambda z: z * 1.0, "relu": f.relu, "gelu": lambda z: 0.5 * z * torch.erfc(-z * math.sqrt(0.5)),
        "silu": f.silu,
        "gelu_tanh": lambda z: f.gelu(z, approximate="tanh")}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sum_units(n, dtype):
    piece = 4096 if dtype is F16 else 16384
    return (0.05 * min(n, piece) + 4 + n / piece) * 2.0 ** -23


def sum_error(a, b):
    return sum_units(a.shape[1], a.dtype) * (a.double().abs() @ b.double().abs().T)


def close(got, want, slack):
    h = half_step(got.dtype)
    least = torch.finfo(got.dtype).smallest_normal * h
    err = (got.double() - want).abs()
    bound = (h + 2.0 ** -23) * want.abs() + (1 + h) * slack + least
    assert (err <= bound).all(), (float((err - bound).max()), float((err / bound).max()))


def tensors(tokens, inner, outer, dtype, bias=True, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()

    return (normal(tokens, inner), normal(outer, inner, scale=inner ** -0.5), normal(outer, scale=0.5) if bias else None,
            normal(tokens, outer) if residual else None, normal(tokens, outer))


def check_forward(out, x, w, b, r, act):
    z = x.double() @ w.double().T
    if b is not None:
        z = z + b.double()
    y = ACTS[act](z)
    slack = 1.13 * (sum_error(x, w) + 2.0 ** -23 * z.abs()) + 2.0 ** -20 * torch.maximum(y.abs(), z.abs() / 8)
    close(out, y if r is None else y + r.double(), slack)


SIZES = [(1, 1, 1), (1, 4096, 512), (2, 64, 128), (7, 65, 129), (16, 100, 1000), (17, 1001, 77), (33, 8, 2050),
         (64, 512, 256), (100, 320, 300), (129, 72, 136), (200, 1000, 511), (256, 256, 640), (257, 130, 128),
         (513, 192, 384), (1100, 96, 264)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("act", ACTS)
def test_forward(cuda_device, size, dtype, act):
    x, w, b, r, _ = tensors(*size, dtype)
    check_forward(fused_linear(x, w, b, r, activation=act), x, w, b, r, act)


@pytest.mark.parametrize("size", [(5, 16384, 300), (300, 12345, 260), (1000, 9000, 130), (40, 40000, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_long_sums_of_one_sign(cuda_device, size, dtype):
    x, w, b, r, _ = tensors(*size, dtype)
    x, w = x.abs(), w.abs()
    check_forward(fused_linear(x, w, b, r, activation="relu"), x, w, b, r, "relu")


@pytest.mark.parametrize("size", SIZES + [(3000, 70, 200), (40, 2048, 32000)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_whole_numbers_are_exact(cuda_device, size, dtype):
    # every sum fits the type: a misplaced element shows, whatever the size
    tokens, inner, outer = size
    g = torch.Generator().manual_seed(1)
    x = torch.zeros(tokens, inner)
    w = torch.zeros(outer, inner)
    x.scatter_(1, torch.randint(0, inner, (tokens, 9), generator=g), torch.randint(-3, 4, (tokens, 9), generator=g).float())
    w = torch.randint(-2, 3, (outer, inner), generator=g).float()
    r = torch.randint(-9, 10, (tokens, outer), generator=g).float()
    x, w, r = (t.to(dtype).cuda() for t in (x, w, r))
    assert torch.equal(fused_linear(x, w, None, r).double(), x.double() @ w.double().T + r.double())
    # the gradients' products in the same way: dz whole numbers with few entries a row and column
    keep = torch.zeros(tokens, outer, dtype=torch.bool)
    keep[torch.arange(tokens), torch.randint(0, outer, (tokens,), generator=g)] = True
    gy = torch.where(keep, torch.randint(-3, 4, (tokens, outer), generator=g), 0).to(dtype).cuda()
    x.requires_grad_(), w.requires_grad_()
    gx, gw = torch.autograd.grad(fused_linear(x, w), (x, w), gy)
    assert torch.equal(gx.double(), gy.double() @ w.detach().double())
    if (gy.double().abs().T @ x.detach().double().abs()).max() <= (256 if dtype is BF16 else 2048):
        assert torch.equal(gw.double(), gy.double().T @ x.detach().double())


def check_gradients(grads, gy, x, w, b, act):
    h = half_step(x.dtype)
    z = x.double() @ w.double().T
    if b is not None:
        z = z + b.double()
    z.requires_grad_(True)
    (dz,) = torch.autograd.grad(ACTS[act](z), z, gy.double())
    # the slope's error: its own, and the sum's through the second derivative (at most 1.6)
    e = gy.double().abs() * (2.0 ** -20 + 1.6 * (sum_error(x, w) + 2.0 ** -23 * z.detach().abs())) + h * dz.abs()
    e = e + torch.finfo(x.dtype).smallest_normal * h        # dz below the normal numbers
    m, n = dz.abs() + e, None
    gx, gw, gb = grads
    if act == "relu":      # the slope jumps at 0
        near = z.detach().abs() <= sum_error(x, w) + 2.0 ** -23 * z.detach().abs()
        e = e + torch.where(near, gy.double().abs(), 0.0)
        m = dz.abs() + e
    for got, a, c in ((gx, dz, w.double().T), (gw, dz.T, x.double().T)):
        if got is None:
            continue
        ea = e if a is dz else e.T
        ma = m if a is dz else m.T
        n = a.shape[1]
        acc = sum_units(n, x.dtype)
        want = a @ c.T
        close(got, want, (ea + acc * ma) @ c.abs().T)
        if act != "relu" and want.norm() > 0 and got.numel() > 50:
            assert float((got.double() - want).norm() / want.norm()) < h
    if gb is not None:
        eb = gy.double().abs() * (2.0 ** -20 + 1.6 * (sum_error(x, w) + 2.0 ** -23 * z.detach().abs()))
        if act == "relu":
            eb = eb + torch.where(near, gy.double().abs(), 0.0)
        close(gb, dz.sum(0), eb.sum(0) + (64 + dz.shape[0] / 64 + 10) * 2.0 ** -24 * m.sum(0))


@pytest.mark.parametrize("size", SIZES + [(2500, 40, 72), (5000, 130, 130)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("act", ACTS)
def test_gradients(cuda_device, size, dtype, act):
    x, w, b, r, gy = tensors(*size, dtype, seed=3)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    out = fused_linear(*leaves, activation=act)
    check_forward(out.detach(), x.detach(), w.detach(), b.detach(), r.detach(), act)
    gx, gw, gb, gr = torch.autograd.grad(out, leaves, gy)
    assert torch.equal(gr, gy)
    check_gradients((gx, gw, gb), gy, x.detach(), w.detach(), b.detach(), act)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences(cuda_device, act):
    # along one direction in each input, from results in 64 bits of the definition at x +- d; the
    # kernel's gradient must predict the difference: second order in d, and the gradients' rounding
    x, w, b, r, gy = tensors(20, 48, 40, F16, seed=5)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(fused_linear(*leaves, r, activation=act), leaves, gy)
    value = lambda x, w, b: float((ACTS[act](x @ w.T + b) * gy.double()).sum())  # noqa: E731
    for i, (t, g) in enumerate(zip(leaves, grads)):
        u = torch.randn(t.shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        step = 1e-5
        moved = [[s.detach().double() + (k * step * u if s is t else 0) for s in leaves] for k in (1, -1)]
        slope = (value(*moved[0]) - value(*moved[1])) / (2 * step)
        # the gradients' error is below h of their norm, independent of u: h |g| |u| by Cauchy's inequality
        assert abs(float((g.double() * u).sum()) - slope) <= half_step(F16) * float(g.double().norm() * u.norm()) + 1e-6


def test_some_gradients(cuda_device):
    x, w, b, r, gy = tensors(37, 100, 60, BF16, seed=7)
    whole = torch.autograd.grad(fused_linear(*[t.requires_grad_() for t in (x, w, b, r)], activation="silu"),
                                (x, w, b, r), gy)
    for k in range(4):
        ins = [t.detach() for t in (x, w, b, r)]
        ins[k] = ins[k].clone().requires_grad_()
        (g,) = torch.autograd.grad(fused_linear(*ins, activation="silu"), ins[k], gy)
        assert torch.equal(g, whole[k])
    with torch.no_grad():
        assert not fused_linear(x, w, b, r).requires_grad


def test_expanded_gradient_and_leading_dims(cuda_device):
    x, w, b, r, _ = tensors(24, 40, 56, BF16, seed=8)
    x3, r3 = x.view(2, 3, 4, 40), r.view(2, 3, 4, 56)
    leaves = [t.requires_grad_() for t in (x3, w, b, r3)]
    out = fused_linear(*leaves, activation="gelu")
    assert out.shape == (2, 3, 4, 56)
    grads = torch.autograd.grad(out.sum(), leaves)
    assert [g.shape for g in grads] == [t.shape for t in leaves]
    ones = torch.ones_like(r)
    check_gradients((grads[0].view(24, 40), grads[1], grads[2]), ones, x.detach(), w.detach(), b.detach(), "gelu")
    assert torch.equal(grads[3], torch.ones_like(r3))
    one = fused_linear(x3[0, 0, 0].detach(), w.detach(), b.detach(), r3[0, 0, 0].detach(), activation="gelu")
    assert one.shape == (56,)
    check_forward(one[None], x[:1].detach(), w.detach(), b.detach(), r[:1].detach(), "gelu")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strides(cuda_device, dtype):
    x, w, b, r, gy = tensors(50, 72, 88, dtype, seed=9)
    want = fused_linear(x, w, b, r, activation="silu")
    room = torch.zeros(50, 100, dtype=dtype, device="cuda")
    for lo in (0, 3, 8):
        room[:, lo:lo + 72] = x
        wide = torch.zeros(88, 80 + lo, dtype=dtype, device="cuda")
        wide[:, lo:lo + 72] = w
        rr = torch.zeros(50, 97, dtype=dtype, device="cuda")
        rr[:, 5:93] = r
        assert torch.equal(fused_linear(room[:, lo:lo + 72], wide[:, lo:lo + 72], b, rr[:, 5:93], activation="silu"), want)
    assert torch.equal(fused_linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r.t().contiguous().t(),
                                    activation="silu"), want)
    bb = torch.zeros(176, dtype=dtype, device="cuda")
    bb[::2] = b
    assert torch.equal(fused_linear(x, w, bb[::2], r, activation="silu"), want)
    one = x[:1].expand(50, 72)
    assert torch.equal(fused_linear(one, w, b, activation="silu")[7], fused_linear(x[:1], w, b, activation="silu")[0])


def test_rows_do_not_depend_on_their_neighbours(cuda_device):
    # NaN and infinity stay in their own rows; tiles' rows past the last are not seen
    x, w, b, r, _ = tensors(70, 200, 300, BF16, seed=10)
    want = fused_linear(x, w, b, r, activation="gelu_tanh")
    x = x.clone()
    x[3, 5], x[40, 199] = math.nan, math.inf
    got = fused_linear(x, w, b, r, activation="gelu_tanh")
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[3] = keep[40] = False
    assert torch.equal(got[keep], want[keep]) and got[3].isnan().all()


@pytest.mark.parametrize("act", ACTS)
def test_far_sums(cuda_device, act):
    # sums from -60000 to 60000: no NaN where the definition has none, in either direction
    z = torch.tensor([-6e4, -1000.0, -90.0, -12.0, -1e-3, 0.0, 1e-3, 12.0, 90.0, 1000.0, 6e4]).to(BF16).cuda()
    x = z[:, None].clone().requires_grad_()
    w = torch.ones(1, 1, dtype=BF16, device="cuda")
    y = fused_linear(x, w, activation=act)
    y.backward(torch.ones_like(y))
    zz = z.double().requires_grad_()
    want = ACTS[act](zz)
    (slope,) = torch.autograd.grad(want.sum(), zz)
    close(y.detach()[:, 0], want.detach(), 2.0 ** -20 * want.detach().abs())
    close(x.grad[:, 0], slope, half_step(BF16) * slope.abs() + 2.0 ** -18)


def test_no_tokens(cuda_device):
    x, w, b, r, _ = tensors(0, 16, 24, BF16)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    out = fused_linear(*leaves, activation="silu")
    assert out.shape == (0, 24)
    gx, gw, gb, gr = torch.autograd.grad(out.sum(), leaves)
    assert gx.shape == (0, 16) and (gw == 0).all() and gw.shape == (24, 16) and (gb == 0).all() and gr.shape == (0, 24)


def test_second_derivatives_are_refused(cuda_device):
    x, w, _, _, gy = tensors(4, 8, 8, BF16)
    x.requires_grad_(), w.requires_grad_()
    (g,) = torch.autograd.grad(fused_linear(x, w, activation="silu"), x, gy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_changed_inputs_are_noticed(cuda_device):
    x, w, _, _, gy = tensors(4, 8, 8, BF16)
    w.requires_grad_()
    out = fused_linear(x, w, activation="silu")
    x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(gy)


def test_streams_and_graphs(cuda_device):
    x, w, b, r, gy = tensors(60, 250, 130, BF16, seed=11)      # 250: copied to aligned rows first
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    want = fused_linear(x, w, b, r, activation="silu")
    with torch.cuda.stream(side):
        got = fused_linear(x, w, b, r, activation="silu")
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # a captured step, forward and backward, replayed on other inputs in the same place
    xs, ws, bs, rs = (t.clone().requires_grad_() for t in (x, w, b, r))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(fused_linear(xs, ws, bs, rs, activation="silu"), (xs, ws, bs), gy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_linear(xs, ws, bs, rs, activation="silu")
        grads = torch.autograd.grad(out, (xs, ws, bs), gy)
    for seed in (12, 13):
        new = tensors(60, 250, 130, BF16, seed=seed)
        with torch.no_grad():
            for t, n in zip((xs, ws, bs, rs), new):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        check_forward(out.detach(), *new[:4], "silu")
        check_gradients(grads, gy, new[0], new[1], new[2], "silu")


def test_inputs_written_just_before(cuda_device):
    x, w, b, r, _ = tensors(300, 512, 512, BF16, seed=14)
    for k in range(5):
        y = x * (k + 1)                                     # a kernel that the call follows at once
        v = w * (k + 1)
        check_forward(fused_linear(y, v, b, r), y, v, b, r, "none")


def test_head_block(cuda_device):
    x, w, b, _, _ = tensors(9, 64, 64, BF16, seed=15)
    assert torch.equal(HeadBlock(w, b)(x), fused_linear(x, w, b, x, activation="silu"))
    assert torch.equal(HeadBlock(w, residual=False, activation="relu")(x), fused_linear(x, w, activation="relu"))


def test_same_bits_every_time(cuda_device):
    x, w, b, r, gy = tensors(900, 300, 400, F16, seed=16)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    first = None
    for _ in range(3):
        out = fused_linear(*leaves, activation="gelu")
        got = [out.detach(), *torch.autograd.grad(out, leaves, gy)]
        assert first is None or all(torch.equal(a, c) for a, c in zip(got, first))
        first = got


def test_from_another_thread(cuda_device):
    # a thread that has not used the device yet
    import threading
    from flashgen_b200 import AdapterHead
    x, w, b, _, _ = tensors(9, 64, 64, BF16, seed=17)
    got = []
    for call in (lambda: fused_linear(x, w, b), lambda: AdapterHead(w).logits(x)):
        t = threading.Thread(target=lambda: got.append(call()))
        t.start()
        t.join()
    assert torch.equal(got[0], fused_linear(x, w, b)) and torch.equal(got[1], AdapterHead(w).logits(x))
