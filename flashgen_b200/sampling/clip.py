"""The global norm of a list of gradients, and clipping to a given norm.

What a training step does between the backward pass (of
:func:`~flashgen_b200.sampling.logprobs.logprobs_and_entropy`, of
:func:`~flashgen_b200.sampling.linear.fused_linear`) and the optimizer. A
sampler-only engine has no counterpart (FlashGen does not train). All tensors
go through two kernel launches of the C ABI (``fg_clip_grad_norm``) on the
current stream, with no host copy and no synchronisation.
"""
from __future__ import annotations

import array
import math
from itertools import chain, repeat
from operator import attrgetter
from typing import List, Optional, Sequence, Union

import torch

from .. import _lib
from .sampler import _DTYPES, _call

# Lists are gone through by map: a training step has hundreds of tensors, and what Python does
# for each of them takes longer than the kernels do.
_dtype, _layout, _shape = attrgetter("dtype"), attrgetter("layout"), attrgetter("shape")
_address, _count, _device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
_dense, _inference = torch.Tensor.is_contiguous, torch.Tensor.is_inference


def _list(tensors: Union[torch.Tensor, Sequence[torch.Tensor]], what: str) -> List[torch.Tensor]:
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    try:
        if set(map(_layout, tensors)) <= {torch.strided} and set(map(_dtype, tensors)) <= _DTYPES.keys():
            return tensors
    except AttributeError:
        pass
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} must be tensors, got {type(t).__name__}")
        if t.layout is not torch.strided or t.dtype not in _DTYPES:
            raise TypeError(f"{what} must be dense float32, float16 or bfloat16 tensors, got {t.layout} {t.dtype}")
    return tensors


def _norm(grads: List[torch.Tensor], out: Optional[List[torch.Tensor]], max_norm: float, scale: float) -> torch.Tensor:
    """One fg_clip_grad_norm call on contiguous tensors."""
    dev = grads[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"flashgen_b200 runs on the GPU only; the gradients are on {dev}")
    devices = set(map(_device, grads if out is None else grads + out))
    if devices != {dev.index}:
        raise ValueError(f"gradients on devices {sorted(devices)}: one call works on one device")
    n = len(grads)
    code = _DTYPES.__getitem__
    codes = map(code, map(_dtype, grads))
    if out is None:
        fields = zip(map(_address, grads), repeat(0), map(_count, grads), codes)
    else:
        both = [g | o << 32 for g, o in zip(codes, map(code, map(_dtype, out)))]
        fields = zip(map(_address, grads), map(_address, out), map(_count, grads), both)
    table = array.array("q", list(chain.from_iterable(fields)))       # FgGradTensor, field by field
    lib = _lib.load()
    need = lib.fg_clip_workspace_size(n)
    if need == 0:
        raise ValueError(f"too many tensors: {n}")
    # (the norm is not a part of the workspace: a caller that keeps it would keep all of that)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    room = torch.empty(need, dtype=torch.uint8, device=dev)
    a = _lib.FgClipArgs(table.buffer_info()[0], n, 0, max_norm, scale, norm.data_ptr(), room.data_ptr(), need)
    _call(dev, lib.fg_clip_grad_norm, a, "fg_clip_grad_norm")
    return norm


def grad_norm(grads: Union[torch.Tensor, Sequence[torch.Tensor]], *, scale: float = 1.0) -> torch.Tensor:
    """``scale * sqrt(sum of squares)`` over all elements of ``grads`` (a tensor or a
    list of them, float32, float16 and bfloat16 mixed as they come), as a float32
    scalar on their device. Summed in 64 bits; neither huge nor tiny gradients
    overflow or vanish on the way. A number for logs and for clipping: no gradient
    flows through it."""
    grads = _list(grads, "grads")
    if not grads:
        raise ValueError("no gradients")
    scale = float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    with torch.no_grad():
        return _norm([g.contiguous() for g in grads], None, math.inf, scale)


def clip_grad_norm(grads: Union[torch.Tensor, Sequence[torch.Tensor]], max_norm: float, *, scale: float = 1.0,
                   out: Union[None, torch.Tensor, Sequence[torch.Tensor]] = None,
                   check_errors: bool = False) -> torch.Tensor:
    """Scale ``grads`` by ``scale * min(1, max_norm / (norm + 1e-6))`` and return
    their ``norm`` before clipping (``scale`` times the root of the sum of
    squares; float32, on their device). ``scale`` undoes a loss scale.

    In place, or into ``out``: tensors of the gradients' shapes, any of the three
    types each, that share no memory with the list. A list that names a tensor
    (or a part of it) twice is refused where it would be written twice. With a
    norm that is NaN every gradient becomes NaN; with an infinite one (of an infinite
    gradient, or above the largest float32) finite gradients become 0, unless
    ``max_norm`` is infinite too: then nothing is clipped. ``check_errors`` reads the
    norm back and raises for both.

    >>> norm = clip_grad_norm([p.grad for p in params if p.grad is not None], 1.0)
    """
    grads = _list(grads, "grads")
    if not grads:
        raise ValueError("no gradients")
    max_norm, scale = float(max_norm), float(scale)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    given = grads if out is None else _list(out, "out")
    if len(given) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(given)} results")
    if out is not None and list(map(_shape, grads)) != list(map(_shape, given)):
        g, o = next((g, o) for g, o in zip(grads, given) if g.shape != o.shape)
        raise ValueError(f"out must have the gradients' shapes, got {tuple(o.shape)} for {tuple(g.shape)}")
    with torch.no_grad():
        src, dst = grads, given
        if not all(map(_dense, grads if out is None else grads + given)):
            # others go through a dense copy, and the results back through one
            src = [g.contiguous() for g in grads]
            dst = [s if o is g else o if o.is_contiguous() else torch.empty_like(o, memory_format=torch.contiguous_format)
                   for g, s, o in zip(grads, src, given)]
            _apart(given)
        norm = _norm(src, dst, max_norm, scale)
        written = given
        if dst is not given:
            written = [o for o, d in zip(given, dst) if o is d]
            for o, d in zip(given, dst):
                if o is not d:
                    o.copy_(d)
        # a graph that saved one of them raises instead of going on with what it finds there
        if any(map(_inference, written)):
            written = [t for t in written if not t.is_inference()]
        torch.autograd.graph.increment_version(written)
    if check_errors and not math.isfinite(float(norm)):
        raise RuntimeError(f"the gradients' norm is {float(norm)}")
    return norm


def _apart(tensors: List[torch.Tensor]) -> None:
    """Refuse results that share memory: through dense copies the library would not see it."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.element_size() *
                    (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in tensors if t.numel())
    for (_, end), (start, _) in zip(spans, spans[1:]):
        if start < end:
            raise ValueError("results that share memory (or lie in each other's gaps) cannot be written in one call")
    for t in tensors:
        if any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
            raise ValueError("a result with expanded dimensions cannot be written")
