"""The dense block in front of an LM head, fused: ``act(x W^T + bias) + residual``.

Decoders put such blocks between the last hidden states and the head (the head
transform of masked models, the residual block of a draft head). FlashGen runs
them as a library product and a kernel each for bias, activation and addition
(csrc/runtime/transformer.cu). :func:`fused_linear` is one kernel launch of the
C ABI (``fg_linear``) whose epilogue does the rest, differentiable through
``fg_linear_grad``; :class:`HeadBlock` keeps a block's parameters for
``DecodeBatch.step_hidden``.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib
from .sampler import _DTYPES, _call, _ptr

_ACTIVATIONS = {"none": _lib.FG_ACT_NONE, "relu": _lib.FG_ACT_RELU, "gelu": _lib.FG_ACT_GELU,
                "gelu_tanh": _lib.FG_ACT_GELU_TANH, "silu": _lib.FG_ACT_SILU}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix as the kernels read it: rows of neighbouring elements that do not overlap."""
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _stride(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
             act: int, keep: bool):
    """The block on matrices. With `keep` also what the gradients read: x and the weight, each as a
    matrix (place None) or as the aligned copy that the call made (the workspace, and the copy's
    place in it: byte offset and stride), and the sums before the activation, in fp32 (the slope
    at a rounded sum would lose its last bits)."""
    tokens, inner, outer = x.shape[0], x.shape[1], weight.shape[0]
    out = x.new_empty((tokens, outer))
    preact = x.new_empty((tokens, (outer + 3) // 4 * 4), dtype=torch.float32) if keep and act else None
    if tokens == 0:
        return out, (x, None), (weight, None), preact
    x, weight = _rows(x), _rows(weight)
    xs, ws = _stride(x), _stride(weight)
    xp, wp = x.data_ptr(), weight.data_ptr()
    lib = _lib.load()
    a = _lib.FgLinearArgs(xp, wp, _ptr(bias), _ptr(residual), out.data_ptr(), _ptr(preact),
                          None, 0, _DTYPES[x.dtype], tokens, inner, outer, act, 0, xs, ws,
                          _stride(residual), outer, _stride(preact))
    # rows on 16-byte boundaries are read where they lie
    copy_x, copy_w = xp % 16 != 0 or (tokens > 1 and xs % 8 != 0), wp % 16 != 0 or (outer > 1 and ws % 8 != 0)
    room = None
    if copy_x or copy_w:
        room = torch.empty(lib.fg_linear_workspace_size(a), dtype=torch.uint8, device=x.device)
        a.workspace, a.workspace_bytes = room.data_ptr(), room.numel()
    _call(x.device, lib.fg_linear, a, "fg_linear")
    if not keep:
        return out, None, None, None
    # the workspace has x's copy, if one was made, then the weight's: rows of inner rounded up to 8
    width = (inner + 7) // 8 * 8
    x_read = (room, (0, width)) if copy_x else (x, None)
    w_read = (room, ((2 * tokens * width + 255) // 256 * 256 if copy_x else 0, width)) if copy_w else (weight, None)
    return out, x_read, w_read, preact


class _Once(torch.autograd.Function):
    """A gradient that is linked to what it was computed from: a backward pass
    through it raises."""

    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("fused_linear is differentiable once: its gradients have no gradients")


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        out, x_read, w_read, preact = _forward(x, weight, bias, residual, act, any(ctx.needs_input_grad[:3]))
        if x_read is not None:
            # (the inputs themselves as well: a change of them before the backward pass is noticed)
            ctx.save_for_backward(x, weight, None if x_read[0] is x else x_read[0],
                                  None if w_read[0] is weight else w_read[0], preact)
            ctx.places, ctx.sizes = (x_read[1], w_read[1]), (*x.shape, weight.shape[0])
        ctx.act = act
        return out

    @staticmethod
    def backward(ctx, grad):
        wanted = ctx.needs_input_grad
        gx = gw = gb = None
        if any(wanted[:3]):
            x, weight, x_read, w_read, preact = ctx.saved_tensors
            gx, gw, gb = _gradients(grad.detach(), x if x_read is None else x_read,
                                    weight if w_read is None else w_read, ctx.places, preact, ctx.sizes, ctx.act, wanted)
            if torch.is_grad_enabled():   # create_graph=True
                gx, gw, gb = (None if g is None else _Once.apply(g, grad, x, weight) for g in (gx, gw, gb))
        return gx, gw, gb, grad if wanted[3] else None, None


def _saved(t: torch.Tensor, place, rows: int, cols: int, dev: int, dtype: torch.dtype):
    """What forward saved, as it came back, with its address and row stride. Hooks on saved tensors
    (offloading) owe the values only: a slice of a wider buffer may come back dense, so nothing
    that was noted of its layout holds. A workspace is a vector of bytes, where places hold."""
    shape = t.shape
    if place is not None:
        if t.dtype is not torch.uint8 or t.get_device() != dev or len(shape) != 1 or shape[0] < place[0] + 2 * rows * place[1]:
            raise RuntimeError(f"a saved workspace came back as {list(shape)} {t.dtype} on {t.device}")
        t = t.contiguous()
        return t, t.data_ptr() + place[0], place[1]
    if t.dtype is not dtype or t.get_device() != dev or shape != (rows, cols):
        raise RuntimeError(f"a saved tensor of {[rows, cols]} {dtype} came back as {list(shape)} {t.dtype} on {t.device}")
    t = _rows(t)
    return t, t.data_ptr(), _stride(t)


def _gradients(grad, x, weight, places, preact, sizes, act, wanted):
    tokens, inner, outer = sizes
    dtype, dev = grad.dtype, grad.device
    gx = torch.empty((tokens, inner), dtype=dtype, device=dev) if wanted[0] else None
    gw = torch.empty((outer, inner), dtype=dtype, device=dev) if wanted[1] else None
    gb = torch.empty((outer,), dtype=dtype, device=dev) if wanted[2] else None
    if tokens == 0:      # sums over nothing
        for g in (gw, gb):
            if g is not None:
                g.zero_()
        return gx, gw, gb
    g, on = _rows(grad), grad.get_device()
    x, xp, xs = _saved(x, places[0], tokens, inner, on, dtype)
    weight, wp, ws = _saved(weight, places[1], outer, inner, on, dtype)
    zp = zs = 0
    if preact is not None:
        preact, zp, zs = _saved(preact, None, tokens, (outer + 3) // 4 * 4, on, torch.float32)
    lib = _lib.load()
    a = _lib.FgLinearGradArgs(
        g.data_ptr(), xp, wp, zp, _ptr(gx), _ptr(gw), _ptr(gb), None, 0, _DTYPES[dtype], tokens, inner, outer, act, 0,
        _stride(g), xs, ws, zs, inner, inner)
    size = lib.fg_linear_grad_workspace_size(a)
    if size:
        room = torch.empty(size, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = room.data_ptr(), size
    _call(dev, lib.fg_linear_grad, a, "fg_linear_grad")
    return gx, gw, gb


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None, *, activation: str = "none") -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: ``x`` [..., inner], ``weight`` [outer,
    inner], ``bias`` [outer], ``residual`` of the result's shape [..., outer], all
    float16 or all bfloat16; ``activation`` is "none", "relu", "gelu" (erf),
    "gelu_tanh" or "silu". Products are summed in fp32, and bias, activation and
    residual are applied to the fp32 sum, which is rounded once.

    Differentiable with respect to all four (once: a second derivative raises, and so
    does a tangent of forward mode).
    For that the sums before the activation are kept in fp32, and their
    gradients enter the two products of the backward pass rounded to the
    operands' type: twice the rounding of a result in the gradients of ``x`` and
    ``weight`` (1.4 times the error), and infinity where one is above 65504 in
    float16.

    A step can be captured into a CUDA graph, forward and backward together, from
    leaves that no graph of an uncaptured step is alive for: autograd would tie the
    captured backward pass to that step's stream, which ends the capture and may
    end the process. Drop such results first, or capture from fresh leaves.

    ``x`` and ``weight`` are read where they lie when their rows are 16-byte
    aligned (``inner`` a multiple of 8, as a rule); otherwise each call copies
    them.

    >>> y = fused_linear(hidden, weight, bias, hidden, activation="silu")
    """
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [outer, inner], got {tuple(weight.shape)}")
    outer, inner = weight.shape
    if x.dim() < 1 or x.shape[-1] != inner:
        raise ValueError(f"x must be [..., {inner}], got {tuple(x.shape)}")
    dtype, dev = weight.dtype, weight.device
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"weight must be float16 or bfloat16, got {dtype}")
    shape = x.shape[:-1] + (outer,)
    for t, what, want in ((x, "x", x.shape), (bias, "bias", (outer,)), (residual, "residual", shape)):
        if t is None:
            continue
        if t.dtype != dtype or t.device != dev:
            raise TypeError(f"{what} must be {dtype} on {dev} like the weight, got {t.dtype} on {t.device}")
        if t.shape != want:
            raise ValueError(f"{what} must be {list(want)}, got {list(t.shape)}")
    # (level below 0: no forward-mode pass is open, the usual case)
    if forward_ad._current_level >= 0:
        for t, what in ((x, "x"), (weight, "weight"), (bias, "bias"), (residual, "residual")):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"fused_linear has no forward-mode derivative; {what} carries a tangent")
    if not weight.is_cuda:
        raise RuntimeError(f"flashgen_b200 runs on the GPU only; the weight is on {dev}")
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, inner)
    r2 = residual if residual is None or flat else residual.reshape(-1, outer)
    if r2 is not None:
        r2 = _rows(r2)
    if bias is not None:
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        out = _FusedLinear.apply(x2, weight, bias, r2, act)
    else:
        out = _forward(x2, weight, bias, r2, act, False)[0]
    return out if flat else out.view(shape)


class HeadBlock:
    """A dense block with its parameters: ``hidden + act(hidden W^T + bias)``, or
    without the first term.

    >>> block = HeadBlock(weight, bias, activation="silu")   # weight [dim, dim]
    >>> ids = dec.step_hidden(hidden, head, block=block)
    """

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "silu",
                 residual: bool = True):
        if weight.dim() != 2 or (residual and weight.shape[0] != weight.shape[1]):
            raise ValueError(f"weight must be [outer, inner], square with a residual, got {tuple(weight.shape)}")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
        self.weight, self.bias, self.activation, self.residual = weight, bias, activation, bool(residual)

    def __call__(self, hidden: torch.Tensor) -> torch.Tensor:
        return fused_linear(hidden, self.weight, self.bias, hidden if self.residual else None,
                            activation=self.activation)
