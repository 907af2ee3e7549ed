"""LM head shared by a batch of requests, each with its own low-rank adapter.

FlashGen's engines compute the logits the sampler reads with one library
product per step (csrc/runtime/transformer.cu:384-389); requests that bring
their own fine-tuned head would need a step each. :class:`AdapterHead` keeps
the shared weight and a bank of adapters on the GPU and computes a whole
batch's logits with one ``fg_adapter_logits`` call, every row with its own
adapter (or none).
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .sampler import _DTYPES, _call, _ptr, _status_error, _written


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    """A [rows, dim] matrix as the kernels read it: 16-byte aligned rows."""
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1] and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    rows, dim = t.shape
    room = torch.zeros(rows, (dim + 7) // 8 * 8, dtype=t.dtype, device=t.device)
    room[:, :dim] = t
    return room[:, :dim]


class AdapterHead:
    """``logits[b] = hidden[b] @ weight.T + scale_a * (hidden[b] @ down_a.T) @ up_a.T``
    with ``a = adapters[b]`` (no second term for a negative id).

    >>> head = AdapterHead(weight, slots=32, rank=16)    # weight [V, dim], float16 or bfloat16
    >>> head.load(3, down, up, scale=alpha / r)          # down [r, dim], up [V, r], r <= rank
    >>> logits = head.logits(hidden, adapters)           # [B, dim], [B] int32 -> [B, V]

    ``weight`` is used where it lies when its rows are 16-byte aligned: later
    in-place updates of it reach the head. Otherwise (an odd ``dim``, a sliced or
    transposed weight) it is laid out anew once, which takes its memory a second
    time, and the head keeps that snapshot: build a new head after an update.
    Adapters are copied into the bank.
    """

    def __init__(self, weight: torch.Tensor, slots: int = 0, rank: int = 16):
        if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
            raise ValueError(f"weight must be [V, dim], got {tuple(weight.shape)}")
        if weight.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"weight must be float16 or bfloat16, got {weight.dtype}")
        if not weight.is_cuda:
            raise RuntimeError(f"flashgen_b200 runs on the GPU only; the weight is on {weight.device}")
        if slots < 0 or not 1 <= rank <= _lib.FG_ADAPTER_MAX_RANK:
            raise ValueError(f"slots must be >= 0 and rank in [1, {_lib.FG_ADAPTER_MAX_RANK}], "
                             f"got {slots} and {rank}")
        self.weight = _dense_rows(weight.detach())
        self.vocab, self.dim = weight.shape
        self.device, self.dtype = weight.device, weight.dtype
        self.slots, self.rank = int(slots), int(rank)
        self._rank = (self.rank + 7) // 8 * 8             # the bank's rank
        width = (self.dim + 7) // 8 * 8
        # a slot's contents count once its scale is not 0
        self._down = torch.empty(self.slots, self._rank, width, dtype=self.dtype, device=self.device)
        self._up = torch.empty(self.slots, self.vocab, self._rank, dtype=self.dtype, device=self.device)
        self._scales = torch.zeros(self.slots, dtype=torch.float32, device=self.device)

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.slots:
            raise IndexError(f"slot {slot} outside [0, {self.slots})")
        return slot

    @torch.no_grad()
    def load(self, slot: int, down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> None:
        """Put an adapter into ``slot`` (on the current stream): its values, without
        its graph."""
        self._slot(slot)
        r = down.shape[0] if down.dim() == 2 else -1
        if down.dim() != 2 or up.dim() != 2 or not 1 <= r <= self.rank or down.shape[1] != self.dim or \
                up.shape != (self.vocab, r):
            raise ValueError(f"an adapter of this head is down [r, {self.dim}] and up [{self.vocab}, r] with "
                             f"r <= {self.rank}, got {tuple(down.shape)} and {tuple(up.shape)}")
        if r < self._rank:
            self._down[slot, r:] = 0
            self._up[slot, :, r:] = 0
        self._down[slot, :r, :self.dim] = down
        self._up[slot, :, :r] = up
        self._scales[slot] = float(scale)

    def unload(self, slot: int) -> None:
        """Empty ``slot``: rows that still name it get the shared logits alone."""
        self._scales[self._slot(slot)] = 0.0

    def logits(self, hidden: torch.Tensor, adapters: Optional[torch.Tensor] = None, *,
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
               check_errors: bool = False) -> torch.Tensor:
        """Logits [B, V] of ``hidden`` [B, dim] with every row's adapter
        (``adapters`` [B] int32, negative: none). ``out_dtype`` is the head's
        type (default) or float32. ``check_errors`` reads the row status back
        and raises for slots outside the bank; without it such rows get the
        shared logits alone. (A wait in the kernel that runs out raises, too;
        unchecked, what was not computed is NaN, which the sampler marks.) There is
        no backward pass: a ``hidden`` that requires
        a gradient is refused outside ``torch.no_grad()``."""
        if hidden.dim() != 2 or hidden.shape[1] != self.dim:
            raise ValueError(f"hidden must be [B, {self.dim}], got {tuple(hidden.shape)}")
        if hidden.dtype != self.dtype or hidden.device != self.device:
            raise TypeError(f"hidden must be {self.dtype} on {self.device}, got {hidden.dtype} on {hidden.device}")
        if hidden.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("AdapterHead.logits has no backward pass: detach hidden or call it under torch.no_grad()")
        B = hidden.shape[0]
        if hidden.stride(1) != 1 or (B > 1 and hidden.stride(0) < self.dim):
            hidden = hidden.contiguous()
        if adapters is not None:
            if adapters.shape != (B,) or adapters.dtype != torch.int32 or adapters.device != self.device:
                raise ValueError(f"adapters must be int32 [{B}] on {self.device}, got {adapters.dtype} "
                                 f"{tuple(adapters.shape)} on {adapters.device}")
            adapters = adapters.contiguous()
        given = out is not None
        if not given:
            out_dtype = self.dtype if out_dtype is None else out_dtype
            if out_dtype not in (self.dtype, torch.float32):
                raise TypeError(f"out_dtype must be {self.dtype} or float32, got {out_dtype}")
            out = hidden.new_empty((B, self.vocab), dtype=out_dtype)
        elif out.shape != (B, self.vocab) or out.dtype not in (self.dtype, torch.float32) or \
                out.device != self.device or out.stride(1) != 1 or (B > 1 and out.stride(0) < self.vocab):
            raise ValueError(f"out must be a row-major {self.dtype} or float32 [{B}, {self.vocab}] on {self.device}")
        if B == 0:
            return out
        lib = _lib.load()
        slots = self.slots if adapters is not None else 0
        need = lib.fg_adapter_workspace_size(B, self.dim, self._rank, slots)
        ws = hidden.new_empty(need, dtype=torch.uint8)
        status = torch.empty(B, dtype=torch.int32, device=self.device) if check_errors else None
        a = _lib.FgAdapterArgs(
            hidden.data_ptr(), self.weight.data_ptr(), self._down.data_ptr() or None, self._up.data_ptr() or None,
            self._scales.data_ptr() or None, _ptr(adapters), out.data_ptr(), _ptr(status), ws.data_ptr(), need,
            _DTYPES[self.dtype], _DTYPES[out.dtype], B, self.dim, self.vocab, self._rank, slots, 0,
            hidden.stride(0) if B > 1 else self.dim, self.weight.stride(0), self._down.stride(1),
            out.stride(0) if B > 1 else self.vocab)
        _call(self.device, lib.fg_adapter_logits, a, "fg_adapter_logits")
        if given:
            _written(out)
        if check_errors:
            msg = _status_error(status)
            if msg is not None:
                raise RuntimeError(msg)
        return out
