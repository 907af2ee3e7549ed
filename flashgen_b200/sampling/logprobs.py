"""Log probabilities of given tokens, with entropy, rank and top alternatives.

What a serving API returns beside each drawn id and what a trainer needs to
rescore rollouts. FlashGen declares the field and never fills it
(``CompletionOutput.cumulative_logprob``, flashgen/outputs.py:25). Every
function is one kernel launch through the C ABI (``fg_token_logprobs``,
``fg_token_logprobs_grad``) on the current stream, with no host copy and no
synchronisation.

The normaliser is kept as two numbers per row, the largest logit and the log
of the sum of ``exp((x - max) / T)``, so that neither large logits nor rows
masked with the type's lowest value cost precision.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib
from .sampler import _DTYPES, _call, _ptr, _row_logits, _status_error, _written


class TokenLogprobs(NamedTuple):
    """Per-row results of :func:`token_logprobs` (device tensors)."""

    logprobs: torch.Tensor                   # [B] float32; 0 where the row has no token
    entropy: torch.Tensor                    # [B] float32
    max: torch.Tensor                        # [B] float32: the largest logit
    logsum: torch.Tensor                     # [B] float32: log sum exp((x - max) / T)
    rank: torch.Tensor                       # [B] int32: ids ahead of the token; -1 without one
    status: torch.Tensor                     # [B] int32: FG_ROW_* bits
    top_ids: Optional[torch.Tensor]          # [B, top] int64, likeliest first (ties: smaller id first)
    top_logprobs: Optional[torch.Tensor]     # [B, top] float32


def _rows(logits: torch.Tensor, what: str) -> torch.Tensor:
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{what} must be [B, V] with V >= 1, got {tuple(logits.shape)}")
    if not logits.is_cuda:
        raise RuntimeError(f"flashgen_b200 runs on the GPU only; {what} are on {logits.device}")
    logits = _row_logits(logits)
    if logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]:   # rows that share memory (expand)
        logits = logits.contiguous()
    return logits


def _vector(t: Optional[torch.Tensor], dtype: torch.dtype, shape: torch.Size, device: int,
            what: str) -> Optional[torch.Tensor]:
    """A per-row vector as the kernels read it: dense, of the rows' ``shape`` ([B]) on their device."""
    if t is None:
        return None
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t
    if t.shape != shape:
        raise ValueError(f"{what} must be [{shape[0]}], got {tuple(t.shape)}")
    if t.get_device() != device:
        raise ValueError(f"{what} are on {t.device}, the logits on cuda:{device}")
    if t.dtype != dtype:
        if t.dtype.is_floating_point != dtype.is_floating_point:
            raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
        t = t.to(dtype)
    return t.contiguous()


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *,
                   temperature: Optional[torch.Tensor] = None, top: int = 0,
                   check_errors: bool = False) -> TokenLogprobs:
    """Log probabilities of ``tokens`` ([B] int64; negative: no token) under
    ``logits`` ([B, V], float32, float16 or bfloat16) at ``temperature`` ([B],
    default 1), the rows' entropies, the tokens' ranks (0: likeliest) and the
    ``top`` likeliest ids (0 to 32) with their log probabilities. All
    statistics are float32 whatever the logits' type. ``check_errors`` reads
    the status back and raises for NaN, +inf or fully masked rows, bad
    temperatures and tokens outside the vocabulary; without it such rows are
    marked in ``status``. The results carry no gradient:
    :func:`logprobs_and_entropy` is the differentiable form.

    >>> r = token_logprobs(logits, ids, top=5)
    >>> r.logprobs, r.top_ids, r.top_logprobs
    """
    logits = _rows(logits, "logits")
    B, V = logits.shape
    shape, index = logits.shape[:1], logits.get_device()
    top = int(top)
    if not 0 <= top <= _lib.FG_LOGPROB_MAX_TOP:
        raise ValueError(f"top must be in [0, {_lib.FG_LOGPROB_MAX_TOP}], got {top}")
    tokens = _vector(tokens, torch.int64, shape, index, "tokens")
    temperature = _vector(temperature, torch.float32, shape, index, "temperature")
    dev = logits.device
    logprobs, entropy, peak, logsum, rank, status = logits.new_empty((6, B), dtype=torch.float32).unbind(0)
    rank, status = rank.view(torch.int32), status.view(torch.int32)
    top_ids = top_lp = None
    if top > 0:
        top_ids = logits.new_empty((B, top), dtype=torch.int64)
        top_lp = logits.new_empty((B, top), dtype=torch.float32)
    if B > 0:
        a = _lib.FgLogprobArgs(
            logits.data_ptr(), _DTYPES[logits.dtype], B, V, top, logits.stride(0) if B > 1 else V,
            _ptr(tokens), _ptr(temperature), logprobs.data_ptr(), entropy.data_ptr(), peak.data_ptr(),
            logsum.data_ptr(), rank.data_ptr(), _ptr(top_ids), _ptr(top_lp), status.data_ptr())
        _call(dev, _lib.load().fg_token_logprobs, a, "fg_token_logprobs")
        if check_errors:
            msg = _status_error(status)
            if msg is not None:
                raise RuntimeError(msg)
    return TokenLogprobs(logprobs, entropy, peak, logsum, rank, status, top_ids, top_lp)


def token_logprobs_grad(logits: torch.Tensor, tokens: Optional[torch.Tensor], max: torch.Tensor,
                        logsum: torch.Tensor, grad_logprobs: Optional[torch.Tensor], *,
                        entropy: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                        temperature: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient with respect to ``logits`` of ``sum(grad_logprobs * logprobs) +
    sum(grad_entropy * entropy)``, from the forward call's ``max``, ``logsum``
    and (with ``grad_entropy``) ``entropy``. The result has the logits' type.
    ``out`` may be ``logits`` itself: the gradient then replaces the logits (a
    graph that saved them raises when it goes back through them). One that
    shares memory with a part of them is refused."""
    rows = _rows(logits, "logits")
    B, V = rows.shape
    shape, index = rows.shape[:1], rows.get_device()
    tokens = _vector(tokens, torch.int64, shape, index, "tokens")
    temperature = _vector(temperature, torch.float32, shape, index, "temperature")
    max = _vector(max, torch.float32, shape, index, "max")
    logsum = _vector(logsum, torch.float32, shape, index, "logsum")
    grad_logprobs = _vector(grad_logprobs, torch.float32, shape, index, "grad_logprobs")
    grad_entropy = _vector(grad_entropy, torch.float32, shape, index, "grad_entropy")
    if grad_entropy is not None and entropy is None:
        raise ValueError("grad_entropy needs the forward call's entropy")
    entropy = _vector(entropy, torch.float32, shape, index, "entropy")
    given = out is not None
    if not given:
        out = rows.new_empty((B, V))
    elif out.shape != rows.shape or out.dtype != rows.dtype or out.device != rows.device or \
            out.stride(1) != 1 or (B > 1 and out.stride(0) < V):
        raise ValueError(f"out must be a row-major {rows.dtype} [{B}, {V}] on {rows.device}")
    if B > 0:
        a = _lib.FgLogprobGradArgs(
            rows.data_ptr(), _DTYPES[rows.dtype], B, V, 0, rows.stride(0) if B > 1 else V, _ptr(tokens),
            _ptr(temperature), max.data_ptr(), logsum.data_ptr(), _ptr(entropy), _ptr(grad_logprobs),
            _ptr(grad_entropy), out.data_ptr(), out.stride(0) if B > 1 else V)
        _call(rows.device, _lib.load().fg_token_logprobs_grad, a, "fg_token_logprobs_grad")
        if given:
            _written(out)
    return out


class _Once(torch.autograd.Function):
    """A gradient that is linked to what it was computed from: a backward pass
    through it raises (``once_differentiable`` would not see the saved logits)."""

    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("logprobs_and_entropy is differentiable once: its gradient has no gradient")


class _LogprobsAndEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        r = token_logprobs(logits, tokens, temperature=temperature)
        ctx.save_for_backward(logits, tokens, temperature, r.max, r.logsum, r.entropy)
        ctx.set_materialize_grads(False)
        # the caller may change both in place: neither is a view (set_ shares the memory, of which
        # nothing else is read), and the entropy that is saved stays as it is
        return r.logprobs.new_empty(0).set_(r.logprobs), r.entropy.clone()

    @staticmethod
    def backward(ctx, grad_logprobs, grad_entropy):
        logits, tokens, temperature, peak, logsum, entropy = ctx.saved_tensors
        if grad_logprobs is None and grad_entropy is None:
            return None, None, None
        with torch.no_grad():
            grad = token_logprobs_grad(logits, tokens, peak, logsum, grad_logprobs, entropy=entropy,
                                       grad_entropy=grad_entropy, temperature=temperature).to(logits.dtype)
        if torch.is_grad_enabled():   # create_graph=True
            grad = _Once.apply(grad, logits, grad_logprobs, grad_entropy)
        return grad, None, None


def logprobs_and_entropy(logits: torch.Tensor, tokens: torch.Tensor,
                         temperature: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Differentiable (with respect to ``logits``) log probabilities of
    ``tokens`` and entropies, both [B] float32: the two terms of a
    policy-gradient loss with an entropy bonus. Differentiable once: a second
    derivative raises. There is no gradient with respect to ``temperature``: one
    that requires it is refused.

    >>> lp, h = logprobs_and_entropy(logits, tokens)
    >>> (-(advantage * lp) - 0.01 * h).mean().backward()
    """
    if temperature is not None and temperature.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("logprobs_and_entropy has no gradient with respect to the temperature: detach it, "
                           "or divide the logits by it")
    return _LogprobsAndEntropy.apply(logits, tokens, temperature)
