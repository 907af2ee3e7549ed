"""Sampling with min-p beside penalties, temperature, top-k and top-p.

Min-p keeps the tokens whose probability is at least ``min_p`` times the
likeliest token's; FlashGen's sampler has no such filter
(flashgen/sampling/sampler.py:102-121). It comes before top-k and top-p, so
that these work on the few tokens it leaves. ``SamplingParams.min_p`` reaches
this path through :class:`~flashgen_b200.sampling.sampler.Sampler` and
``DecodeBatch``; :func:`sample_min_p` takes per-row device vectors and also
returns the drawn ids' log probabilities among the tokens that were kept, the
behaviour policy a policy-gradient step needs.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib
from .sampler import _DTYPES, _call, _ptr, _row_logits, _status_error


class MinPSample(NamedTuple):
    """Per-row results of :func:`sample_min_p` (device tensors)."""

    ids: torch.Tensor          # [B] int64; -1 for rows that cannot be sampled
    logprobs: torch.Tensor     # [B] float32: of the id among the kept tokens; 0 for greedy rows
    kept: torch.Tensor         # [B] int32: kept tokens; 1 for greedy rows
    status: torch.Tensor       # [B] int32: FG_ROW_* bits


def _vector(t: Optional[torch.Tensor], dtype: torch.dtype, rows: int, dev: torch.device, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != rows:
        raise ValueError(f"{what} must be [{rows}], got {list(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, the logits on {dev}")
    if t.dtype != dtype:
        if t.dtype.is_floating_point != dtype.is_floating_point:
            raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def sample_min_p(logits: torch.Tensor, uniforms: torch.Tensor, min_p: torch.Tensor, *,
                 temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
                 top_p: Optional[torch.Tensor] = None, greedy: Optional[torch.Tensor] = None,
                 repetition_penalty: Optional[torch.Tensor] = None, presence_penalty: Optional[torch.Tensor] = None,
                 frequency_penalty: Optional[torch.Tensor] = None,
                 history: Optional[Tuple[torch.Tensor, torch.Tensor, int]] = None,
                 check_errors: bool = False) -> MinPSample:
    """Draw one token a row of ``logits`` ([B, V], float32, float16 or bfloat16) with the
    given ``uniforms`` ([B] in [0, 1)): penalties over ``history`` (int32 ids of all rows one
    after the other, int64 offsets [B + 1], the longest row's length), temperature (0:
    greedy), then of the tokens with at least ``min_p`` ([B] in [0, 1]; 0: off) times the
    largest probability the ``top_k`` likeliest (ties kept; <= 0: off), and of those the
    ``top_p`` nucleus. Every parameter is a vector of one value a row. Nothing is copied to
    the host; ``check_errors`` reads the status back and raises. No gradient flows through
    the log probabilities (``logprobs_and_entropy`` has one).

    >>> r = sample_min_p(logits, torch.rand(B, device="cuda"), min_p, temperature=temperature)
    >>> r.ids, r.logprobs
    """
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [B, V] with V >= 1, got {tuple(logits.shape)}")
    if not logits.is_cuda:
        raise RuntimeError(f"flashgen_b200 samples on the GPU only; logits are on {logits.device}")
    logits = _row_logits(logits)
    B, V = logits.shape
    if B > 1 and logits.stride(0) < V:     # rows that share memory (expand)
        logits = logits.contiguous()
    dev, f32 = logits.device, torch.float32
    if uniforms is None or min_p is None:
        raise TypeError("uniforms and min_p must be tensors of one value a row")
    uniforms = _vector(uniforms, f32, B, dev, "uniforms")
    min_p = _vector(min_p, f32, B, dev, "min_p")
    temperature = _vector(temperature, f32, B, dev, "temperature")
    top_p = _vector(top_p, f32, B, dev, "top_p")
    top_k = _vector(top_k, torch.int32, B, dev, "top_k")
    if greedy is not None:
        greedy = _vector(greedy.view(torch.uint8) if greedy.dtype is torch.bool else greedy, torch.uint8, B, dev, "greedy")
    repetition_penalty = _vector(repetition_penalty, f32, B, dev, "repetition_penalty")
    presence_penalty = _vector(presence_penalty, f32, B, dev, "presence_penalty")
    frequency_penalty = _vector(frequency_penalty, f32, B, dev, "frequency_penalty")
    ids = offsets = None
    longest = 0
    if history is not None:
        ids, offsets, longest = history
        longest = int(longest)
        if longest < 0:
            raise ValueError(f"the longest history must be >= 0, got {longest}")
        if ids.dim() != 1:
            raise ValueError(f"history ids must be one vector, got {list(ids.shape)}")
        ids = _vector(ids, torch.int32, ids.shape[0], dev, "history ids")
        offsets = _vector(offsets, torch.int64, B + 1, dev, "history offsets")
        if ids.numel() == 0:
            ids = offsets = None
            longest = 0
        else:
            longest = max(1, longest)
    lib = _lib.load()
    need = lib.fg_sample_min_p_workspace_size(B, V, longest)
    out = torch.empty(B, dtype=torch.int64, device=dev)
    logprobs, kept, status = torch.empty((3, B), dtype=f32, device=dev).unbind(0)
    r = MinPSample(out, logprobs, kept.view(torch.int32), status.view(torch.int32))
    if B == 0:
        return r
    room = torch.empty(need, dtype=torch.uint8, device=dev)
    a = _lib.FgMinPArgs(
        _lib.FgSampleArgs(logits.data_ptr(), _DTYPES[logits.dtype], B, V, longest, logits.stride(0) if B > 1 else V,
                          0, 0, _ptr(ids), _ptr(offsets), _ptr(temperature), _ptr(top_p), _ptr(top_k),
                          _ptr(repetition_penalty), _ptr(presence_penalty), _ptr(frequency_penalty), _ptr(greedy),
                          uniforms.data_ptr(), out.data_ptr(), status.data_ptr(), None, room.data_ptr(), need),
        _ptr(min_p), logprobs.data_ptr(), kept.data_ptr())
    _call(dev, lib.fg_sample_min_p, a, "fg_sample_min_p")
    if check_errors:
        msg = _status_error(r.status)
        if msg is not None:
            raise RuntimeError(msg)
    return r
