"""Outputs that share memory with the inputs they are computed from: refused by the C ABI before anything
runs, unless no row meets another (column slices of one buffer). The addresses are made up, so these tests
run only where there is no GPU: what is not refused ends at the missing device."""
import ctypes
import random

import pytest
import torch

from flashgen_b200 import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses must not reach a device")
BASE = 1 << 20


def _grad(logits, row_stride, out, grad_stride, batch, vocab):
    a = _lib.FgLogprobGradArgs()
    a.logits, a.row_stride, a.out_grad, a.grad_stride = BASE + 2 * logits, row_stride, BASE + 2 * out, grad_stride
    a.dtype, a.batch, a.vocab, a.max, a.logsum = _lib.FG_DTYPE_F16, batch, vocab, 16, 16
    return _lib.load().fg_token_logprobs_grad(ctypes.byref(a), None)


def _meet(a, sa, la, na, b, sb, lb, nb):
    cells = {a + i * sa + k for i in range(na) for k in range(la)}
    return any(b + j * sb + k in cells for j in range(nb) for k in range(lb))


@pytest.mark.parametrize("case", [
    dict(logits=0, row_stride=10, out=1, grad_stride=10, batch=3, vocab=8),        # a column further
    dict(logits=5, row_stride=10, out=0, grad_stride=10, batch=3, vocab=8),
    dict(logits=0, row_stride=8, out=8, grad_stride=8, batch=3, vocab=8),          # a row further
    dict(logits=0, row_stride=20, out=7, grad_stride=20, batch=2, vocab=8),        # the last column
    dict(logits=0, row_stride=8, out=4, grad_stride=16, batch=4, vocab=8)])
def test_gradient_over_part_of_the_logits(case):
    assert _meet(case["logits"], case["row_stride"], case["vocab"], case["batch"],
                 case["out"], case["grad_stride"], case["vocab"], case["batch"])
    assert _grad(**case) == _lib.FG_EINVAL


@pytest.mark.parametrize("case", [
    dict(logits=0, row_stride=10, out=0, grad_stride=10, batch=3, vocab=8),        # the logits themselves
    dict(logits=0, row_stride=16, out=8, grad_stride=16, batch=3, vocab=8),        # column slices of one buffer
    dict(logits=8, row_stride=16, out=0, grad_stride=16, batch=3, vocab=8),
    dict(logits=0, row_stride=8, out=24, grad_stride=8, batch=3, vocab=8)])        # one after the other
def test_gradient_beside_the_logits(case):
    assert _grad(**case) != _lib.FG_EINVAL


def test_gradient_at_random():
    rng = random.Random(0)
    seen = set()
    for _ in range(3000):
        vocab, batch = rng.randint(1, 9), rng.randint(1, 6)
        sa, sb = vocab + rng.randint(0, 12), vocab + rng.randint(0, 12)
        if rng.random() < 0.5:
            sb = sa
        a, b = rng.randint(0, 60), rng.randint(0, 60)
        if a == b:
            continue
        meet = _meet(a, sa, vocab, batch, b, sb, vocab, batch)
        assert (_grad(a, sa, b, sb, batch, vocab) == _lib.FG_EINVAL) == meet, (a, sa, b, sb, vocab, batch)
        seen.add(meet)
    assert seen == {True, False}


def _head(hidden, hidden_stride, out, out_stride, batch, dim, vocab, weight=1 << 24):
    a = _lib.FgAdapterArgs()
    a.hidden, a.out, a.weight = BASE + 2 * hidden, BASE + 2 * out, BASE + 2 * weight
    a.hidden_stride, a.out_stride, a.weight_stride = hidden_stride, out_stride, 64
    a.dtype = a.out_dtype = _lib.FG_DTYPE_BF16
    a.batch, a.dim, a.vocab, a.slots, a.rank = batch, dim, vocab, 0, 16
    a.workspace, a.workspace_bytes = 1 << 30, 1 << 30
    return _lib.load().fg_adapter_logits(ctypes.byref(a), None)


def test_logits_over_hidden_states_or_weight():
    assert _head(0, 100, 40, 100, 3, 50, 60) == _lib.FG_EINVAL          # the last ten columns of a row
    assert _head(0, 110, 50, 110, 3, 50, 60) != _lib.FG_EINVAL          # beside each other in one buffer
    assert _head(0, 50, 100, 60, 3, 50, 60) == _lib.FG_EINVAL           # over the last row
    assert _head(0, 50, 150, 60, 3, 50, 60) != _lib.FG_EINVAL
    assert _head(0, 50, 4096 + 3000, 60, 3, 50, 60, weight=4096) == _lib.FG_EINVAL
    assert _head(0, 50, 4096 + 60 * 64, 60, 3, 50, 60, weight=4096) != _lib.FG_EINVAL
