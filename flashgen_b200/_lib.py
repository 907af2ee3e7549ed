"""ctypes binding of include/flashgen_sampler.h.

The shared library is built in tree by ``flashgen_b200.build``. Loading fails
loudly when it is missing: there is no CPU or PyTorch fallback for sampling.
"""
from __future__ import annotations

import ctypes
import os
import threading

from . import build as _build

FG_OK, FG_EINVAL, FG_ELAUNCH, FG_ENOTSUP, FG_EDEVICE, FG_ESCRATCH = 0, 1, 2, 3, 4, 5
FG_DTYPE_F32, FG_DTYPE_F16, FG_DTYPE_BF16 = 0, 1, 2

FG_ROW_NAN = 0x0001
FG_ROW_POS_INF = 0x0002
FG_ROW_ALL_MASKED = 0x0004
FG_ROW_BAD_HISTORY = 0x0008
FG_ROW_BAD_PARAM = 0x0010
FG_ROW_BAD_UNIFORM = 0x0020
FG_ROW_TIMEOUT = 0x0040
FG_ROW_CAND_TRUNC = 0x0080
FG_ROW_ERROR_MASK = 0x00FF
FG_ROW_GENERAL_PATH = 0x0100
FG_ROW_GREEDY = 0x0200

EXPORTED_SYMBOLS = ("fg_sample", "fg_sample_workspace_size", "fg_sample_candidates", "fg_sample_noalloc",
                    "fg_sample_set_split",
                    "fg_apply_repetition_penalty", "fg_argmax", "fg_token_logprobs", "fg_token_logprobs_grad",
                    "fg_adapter_logits", "fg_adapter_set_wait", "fg_adapter_workspace_size", "fg_strerror", "fg_version")


class FgSampleArgs(ctypes.Structure):
    """Mirror of ``FgSampleArgs`` (field order and types must match the header)."""

    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("batch", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("hist_max_len", ctypes.c_int32),
        ("row_stride", ctypes.c_int64),
        ("vocab_offset", ctypes.c_int64),
        ("vocab_total", ctypes.c_int64),
        ("hist_ids", ctypes.c_void_p),
        ("hist_offsets", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("top_p", ctypes.c_void_p),
        ("top_k", ctypes.c_void_p),
        ("repetition_penalty", ctypes.c_void_p),
        ("presence_penalty", ctypes.c_void_p),
        ("frequency_penalty", ctypes.c_void_p),
        ("greedy", ctypes.c_void_p),
        ("uniforms", ctypes.c_void_p),
        ("out_ids", ctypes.c_void_p),
        ("out_status", ctypes.c_void_p),
        ("out_probs", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class FgLogprobArgs(ctypes.Structure):
    """Mirror of ``FgLogprobArgs``."""

    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("batch", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("top", ctypes.c_int32),
        ("row_stride", ctypes.c_int64),
        ("tokens", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("out_logprobs", ctypes.c_void_p),
        ("out_entropy", ctypes.c_void_p),
        ("out_max", ctypes.c_void_p),
        ("out_logsum", ctypes.c_void_p),
        ("out_rank", ctypes.c_void_p),
        ("out_top_ids", ctypes.c_void_p),
        ("out_top_logprobs", ctypes.c_void_p),
        ("out_status", ctypes.c_void_p),
    ]


class FgLogprobGradArgs(ctypes.Structure):
    """Mirror of ``FgLogprobGradArgs``."""

    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("batch", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("row_stride", ctypes.c_int64),
        ("tokens", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("max", ctypes.c_void_p),
        ("logsum", ctypes.c_void_p),
        ("entropy", ctypes.c_void_p),
        ("grad_logprobs", ctypes.c_void_p),
        ("grad_entropy", ctypes.c_void_p),
        ("out_grad", ctypes.c_void_p),
        ("grad_stride", ctypes.c_int64),
    ]


class FgAdapterArgs(ctypes.Structure):
    """Mirror of ``FgAdapterArgs``."""

    _fields_ = [
        ("hidden", ctypes.c_void_p),
        ("weight", ctypes.c_void_p),
        ("down", ctypes.c_void_p),
        ("up", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("adapters", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("out_status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("batch", ctypes.c_int32),
        ("dim", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("rank", ctypes.c_int32),
        ("slots", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("hidden_stride", ctypes.c_int64),
        ("weight_stride", ctypes.c_int64),
        ("down_stride", ctypes.c_int64),
        ("out_stride", ctypes.c_int64),
    ]


FG_SAMPLE_WORKSPACE_MIN_BYTES = 256
FG_ADAPTER_MAX_RANK = 128
FG_LOGPROB_MAX_TOP = 32


_lib = None
_lock = threading.Lock()


def lib_path() -> str:
    return _build.LIBPATH


def load(build_if_missing: bool = True) -> ctypes.CDLL:
    """Load (building first if needed) the sampler library."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = _build.LIBPATH
        if not os.path.exists(path):
            if not build_if_missing:
                raise RuntimeError(f"flashgen_b200: {path} is missing; run `python -m flashgen_b200.build`")
            _build.build()
        lib = ctypes.CDLL(path)
        lib.fg_sample.argtypes = [ctypes.POINTER(FgSampleArgs), ctypes.c_void_p]
        lib.fg_sample.restype = ctypes.c_int
        lib.fg_sample_workspace_size.argtypes = [ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32]
        lib.fg_sample_workspace_size.restype = ctypes.c_size_t
        lib.fg_sample_candidates.argtypes = [ctypes.POINTER(FgSampleArgs), ctypes.c_void_p, ctypes.c_void_p,
                                             ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p]
        lib.fg_sample_candidates.restype = ctypes.c_int
        lib.fg_sample_noalloc.argtypes = [ctypes.POINTER(FgSampleArgs), ctypes.c_void_p]
        lib.fg_sample_noalloc.restype = ctypes.c_int
        lib.fg_sample_set_split.argtypes = [ctypes.c_int]
        lib.fg_sample_set_split.restype = ctypes.c_int
        lib.fg_apply_repetition_penalty.argtypes = [
            ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int64,
            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
        lib.fg_apply_repetition_penalty.restype = ctypes.c_int
        lib.fg_argmax.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                  ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p]
        lib.fg_argmax.restype = ctypes.c_int
        lib.fg_token_logprobs.argtypes = [ctypes.POINTER(FgLogprobArgs), ctypes.c_void_p]
        lib.fg_token_logprobs.restype = ctypes.c_int
        lib.fg_token_logprobs_grad.argtypes = [ctypes.POINTER(FgLogprobGradArgs), ctypes.c_void_p]
        lib.fg_token_logprobs_grad.restype = ctypes.c_int
        lib.fg_adapter_logits.argtypes = [ctypes.POINTER(FgAdapterArgs), ctypes.c_void_p]
        lib.fg_adapter_logits.restype = ctypes.c_int
        lib.fg_adapter_set_wait.argtypes = [ctypes.c_int64, ctypes.c_int32]
        lib.fg_adapter_set_wait.restype = ctypes.c_int
        lib.fg_adapter_workspace_size.argtypes = [ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32]
        lib.fg_adapter_workspace_size.restype = ctypes.c_size_t
        lib.fg_strerror.argtypes = [ctypes.c_int]
        lib.fg_strerror.restype = ctypes.c_char_p
        lib.fg_version.argtypes = []
        lib.fg_version.restype = ctypes.c_int
        _lib = lib
        return lib


def set_workspace(a: FgSampleArgs, ws) -> None:
    """Point ``a`` at a device workspace tensor and record its size."""
    a.workspace = ws.data_ptr()
    a.workspace_bytes = ws.numel() * ws.element_size()


def workspace_size(batch: int, vocab: int, dtype: int, hist_max_len: int) -> int:
    """Workspace bytes of fg_sample's fastest path for this shape."""
    return int(load().fg_sample_workspace_size(batch, vocab, dtype, max(0, int(hist_max_len))))


def check(rc: int, what: str) -> None:
    if rc != FG_OK:
        msg = load().fg_strerror(rc).decode()
        raise RuntimeError(f"{what} failed: {msg} (code {rc})")
