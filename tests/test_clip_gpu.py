"""The gradient norm and clipping against their definition in 64 bits.

Tolerances: the squares are summed in 64 bits, but for those of one 16-byte vector (up to
eight products added in fp32: 8 roundings of 2^-24, halved by the root), and the norm is
rounded once (2^-24): 5 * 2^-24. A scaled gradient carries the norm's error, the rounding
of norm + 1e-6, of the quotient, of its product with `scale` and of the product with the
gradient (2^-24 each): 9 * 2^-24, and the rounding to its type."""
import math

import pytest
import torch

from flashgen_b200 import clip_grad_norm, grad_norm

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(shapes, dtypes, scale, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(d).cuda() for s, d in zip(shapes, dtypes)]


def norm_of(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def check(grads, before, norm, max_norm, scale=1.0):
    want = norm_of(before) * scale
    assert norm.shape == () and norm.dtype is F32 and norm.device == before[0].device
    assert abs(float(norm) - want) <= 5 * EPS * want
    c = scale * min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        ref = b.double() * c
        half = torch.finfo(g.dtype).eps / 2
        least = torch.finfo(g.dtype).smallest_normal * half      # half a step below the normal numbers
        assert ((g.double() - ref).abs() <= (half + 9 * EPS) * ref.abs() + least).all()


SHAPES = {"one": [(1,)], "few": [(3,), (1025,), (7, 9)], "odd": [(4097,), (1,), (0,), (8191, 3), (2, 5, 7)],
          "chunks": [(16384,), (16385,), (40000,), (8192,)], "many": [(i % 37,) for i in range(400)],
          "large": [(3000, 4001), (5,), (1 << 20,)]}


@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "mixed"])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_in_place(cuda_device, name, kind, max_norm):
    shapes = SHAPES[name]
    kinds = {"f32": [F32], "f16": [F16], "bf16": [BF16], "mixed": [F32, BF16, F16]}[kind]
    grads = make(shapes, [kinds[i % len(kinds)] for i in range(len(shapes))], 1.0)
    before = [g.clone() for g in grads]
    assert abs(float(grad_norm(grads)) - norm_of(before)) <= 5 * EPS * norm_of(before)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    versions = [g._version for g in grads]
    norm = clip_grad_norm(grads, max_norm)
    check(grads, before, norm, max_norm)
    assert all(g._version > v for g, v in zip(grads, versions))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("odtype", [F32, F16, BF16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_out_and_alignment(cuda_device, dtype, odtype, shift):
    before = make([(5000,), (33, 129), (1,)], [dtype] * 3, 0.1)
    rooms = [torch.zeros(b.numel() + 8, dtype=dtype, device="cuda") for b in before]
    grads = [r[shift:shift + b.numel()].view(b.shape).copy_(b) for r, b in zip(rooms, before)]
    outs = [torch.full((b.numel() + 8,), 7.0, dtype=odtype, device="cuda") for b in before]
    out = [o[2 * shift % 5:][:b.numel()].view(b.shape) for o, b in zip(outs, before)]
    norm = clip_grad_norm(grads, 0.25, scale=0.125, out=out)
    check(out, before, norm, 0.25, 0.125)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    for o, b in zip(outs, before):     # nothing written beside the results
        lo = 2 * shift % 5
        assert (o[:lo] == 7).all() and (o[lo + b.numel():] == 7).all()


@pytest.mark.parametrize("size", [1e-30, 1e-23, 1e19, 1e30])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_from_one(cuda_device, size, dtype):
    grads = make([(5000,), (17,)], [dtype] * 2, size) + [torch.zeros(9000, dtype=dtype, device="cuda")]
    before = [g.clone() for g in grads]
    assert abs(float(grad_norm(grads)) - norm_of(before)) <= 5 * EPS * norm_of(before)
    if size > 1:
        check(grads, before, clip_grad_norm(grads, 1.0), 1.0)


def test_a_few_large_among_many_small(cuda_device):
    g = torch.full((1 << 22,), 1e-4, device="cuda")
    g[12345] = 100.0
    want = norm_of([g])
    assert abs(float(grad_norm(g)) - want) <= 5 * EPS * want


def test_not_finite(cuda_device):
    for bad in (math.nan, math.inf):
        grads = make([(100,), (5000,)], [F32, F16], 1.0)
        grads[1][77] = bad
        with pytest.raises(RuntimeError, match="norm is"):
            clip_grad_norm(grads, 1.0, check_errors=True)
        if math.isnan(bad):
            assert all(g.isnan().all() for g in grads)
        else:
            assert grads[1][77].isnan() and (grads[0] == 0).all() and (grads[1].nan_to_num(0.0) == 0).all()


def test_empty_and_infinite_limit(cuda_device):
    empty = [torch.empty(0, device="cuda"), torch.empty(0, 5, dtype=F16, device="cuda")]
    assert float(clip_grad_norm(empty, 1.0)) == 0.0 and float(grad_norm(empty)) == 0.0
    grads = make([(100,)], [F32], 3.0)
    before = grads[0].clone()
    clip_grad_norm(grads, math.inf)
    assert torch.equal(grads[0], before)
    clip_grad_norm(grads, 0.0)
    assert (grads[0] == 0).all()


@pytest.mark.parametrize("count", [96, 97, 700])
def test_many_tensors(cuda_device, count):
    grads = make([(50 + i,) for i in range(count)], [F32] * count, 1.0)
    before = [g.clone() for g in grads]
    check(grads, before, clip_grad_norm(grads, 1.0), 1.0)


def test_strided(cuda_device):
    base = make([(64, 50), (64, 50)], [F32, BF16], 1.0)
    grads = [base[0].t(), base[1][:, 3:40]]
    keep = [b.clone() for b in base]
    before = [g.clone() for g in grads]
    check(grads, before, clip_grad_norm(grads, 1.0), 1.0)
    assert torch.equal(base[1][:, :3], keep[1][:, :3]) and torch.equal(base[1][:, 40:], keep[1][:, 40:])
    out = [torch.zeros(50, 64, device="cuda").t().t(), torch.zeros(37, 64, device="cuda").t()]
    grads = [b.clone() for b in before]
    check(out, before, clip_grad_norm(grads, 1.0, out=out), 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm([base[0].t(), base[0][2:]], 1.0)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm([torch.ones(1, device="cuda").expand(5)], 1.0)


def test_a_tensor_twice(cuda_device):
    g = make([(100,)], [F32], 1.0)[0]
    with pytest.raises(RuntimeError, match="invalid argument"):
        clip_grad_norm([g, g], 1.0)
    with pytest.raises(RuntimeError, match="invalid argument"):
        clip_grad_norm([g, g[50:]], 1.0)
    want = norm_of([g, g])
    assert abs(float(grad_norm([g, g])) - want) <= 5 * EPS * want          # counted twice, written never
    out = [torch.empty_like(g), torch.empty_like(g)]
    check(out, [g, g], clip_grad_norm([g, g], 1.0, out=out), 1.0)


def test_same_bits_every_time(cuda_device):
    grads = make([(100000,), (333,)] * 20, [BF16, F32] * 20, 1.0)
    assert len({float(grad_norm(grads)) for _ in range(5)}) == 1


def test_streams_and_graphs(cuda_device):
    a, b = make([(300000,), (17,)], [F32, BF16], 1.0), make([(200000,)], [F16], 2.0, seed=1)
    keep = [t.clone() for t in a + b]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    norms = [clip_grad_norm(a, 1.0)]
    with torch.cuda.stream(side):
        norms.append(clip_grad_norm(b, 0.5))
    torch.cuda.synchronize()
    check(a, keep[:2], norms[0], 1.0)
    check(b, keep[2:], norms[1], 0.5)
    # captured: replayed on new gradients in the same place
    for t, k in zip(a, keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n1 = clip_grad_norm(a, 1.0)
        n2 = clip_grad_norm(a, 0.5)
    for factor in (1.0, 3.0):
        for t, k in zip(a, keep):
            t.copy_(k * factor)
        before = [t.clone() for t in a]
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(n1) - norm_of(before)) <= 5 * EPS * norm_of(before)
        assert abs(float(n2) - 1.0) < 0.01          # bf16 gradients: what the first clip left
        assert norm_of(a) < 0.51
