"""What the fused linear block's backward pass hands to fg_linear_grad when hooks give the saved
tensors back in another layout: every row that the call describes lies in its tensor (no GPU; the
library's calls are recorded, not made)."""
import ctypes

import pytest
import torch

from flashgen_b200.sampling import linear

BF16 = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(linear, "_call", lambda dev, fn, args, what: made.append((what, args)))
    return made


def sliced(rows, cols, width, lo=0):
    return torch.randn(rows, width).to(BF16)[:, lo:lo + cols]


class Keep:
    """Hooks on saved tensors that give back what `back` makes of them, and remember it."""

    def __init__(self, back):
        self.back, self.tensors = back, []

    def unpack(self, t):
        t = self.back(t)
        self.tensors.append(t)
        return t

    def __enter__(self):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, self.unpack)
        return self.hooks.__enter__()

    def __exit__(self, *e):
        return self.hooks.__exit__(*e)


def dense(t):
    return t.detach().clone(memory_format=torch.contiguous_format)


def wide(t):
    # rows further apart than they were
    if t.dim() != 2:
        return t.detach().clone()
    return torch.cat([t.detach(), torch.zeros_like(t), torch.zeros_like(t)], 1)[:, :t.shape[1]]


def columns_first(t):
    return t.detach().t().contiguous().t() if t.dim() == 2 else t.detach().clone()


@pytest.mark.parametrize("back", [dense, wide, columns_first])
# strided and aligned (read where it lies), strided and not (copied), dense
@pytest.mark.parametrize("x_width,x_lo", [(104, 0), (104, 8), (101, 3), (72, 0)])
@pytest.mark.parametrize("w_width,w_lo", [(80, 0), (75, 1), (72, 0)])
def test_rows_lie_in_their_tensors(calls, back, x_width, x_lo, w_width, w_lo):
    tokens, inner, outer = 50, 72, 88
    x, w = sliced(tokens, inner, x_width, x_lo), sliced(outer, inner, w_width, w_lo)
    x.requires_grad_(), w.requires_grad_()
    keep = Keep(back)
    with keep:
        out = linear._FusedLinear.apply(x, w, None, None, linear._ACTIVATIONS["silu"])
    torch.autograd.grad(out, (x, w), torch.randn(tokens, outer).to(BF16))
    (_, _), (what, a) = calls
    assert what == "fg_linear_grad"
    storages = [(t.untyped_storage().data_ptr(), t.untyped_storage().nbytes()) for t in keep.tensors]

    def room(address):
        at = [lo + n - address for lo, n in storages if lo <= address < lo + n]
        # (a dense copy that the backward pass made itself is no longer there to be looked at)
        return at[0] if at else None

    seen = 0
    for address, stride, rows, cols, size in ((a.x, a.x_stride, tokens, inner, 2), (a.weight, a.weight_stride, outer, inner, 2),
                                              (a.preact, a.preact_stride, tokens, outer, 4)):
        if room(address) is None:
            assert back is columns_first and stride >= cols
            continue
        seen += 1
        assert ((rows - 1) * stride + cols) * size <= room(address), (stride, cols)
    assert seen == 3 or back is columns_first


def test_the_values_of_a_slice(calls):
    # the rows that the call describes are the input's
    x, w = sliced(50, 72, 104, 8), sliced(88, 72, 80)
    x.requires_grad_(), w.requires_grad_()
    keep = Keep(dense)
    with keep:
        out = linear._FusedLinear.apply(x, w, None, None, 0)
    torch.autograd.grad(out, (x, w), torch.randn(50, 88).to(BF16))
    a = calls[-1][1]
    for address, stride, t in ((a.x, a.x_stride, x), (a.weight, a.weight_stride, w)):
        for r in (0, 1, t.shape[0] - 1):
            row = (ctypes.c_int16 * t.shape[1]).from_address(address + 2 * r * stride)
            assert torch.equal(torch.tensor(list(row), dtype=torch.int16), t[r].detach().view(torch.int16))


@pytest.mark.parametrize("back", [lambda t: t.detach().double(), lambda t: t.detach()[:-1], lambda t: t.detach().flatten(),
                                  lambda t: t.detach().half()])
@pytest.mark.parametrize("width", [72, 75])
def test_other_shapes_and_types_are_refused(calls, back, width):
    x, w = sliced(50, 72, width), sliced(88, 72, width)
    x.requires_grad_(), w.requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: back(t)):
        out = linear._FusedLinear.apply(x, w, None, None, linear._ACTIVATIONS["gelu"])
    with pytest.raises(RuntimeError, match="came back as"):
        torch.autograd.grad(out, (x, w), torch.randn(50, 88).to(BF16))
    assert len(calls) == 1
