"""The LM head with adapters: struct layout, workspace size and the C ABI's
refusals, without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

from flashgen_b200 import _lib
from flashgen_b200.sampling.lm_head import AdapterHead

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header(tmp_path):
    cls = _lib.FgAdapterArgs
    fields = [f[0] for f in cls._fields_]
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flashgen_sampler.h"\nint main(void){\n'
    prog += 'printf("%zu\\n", sizeof(FgAdapterArgs));\n'
    for f in fields:
        prog += f'printf("%zu\\n", offsetof(FgAdapterArgs, {f}));\n'
    c = tmp_path / "probe.c"
    c.write_text(prog + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)])
    vals = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert vals[0] == ctypes.sizeof(cls)
    for f, off in zip(fields, vals[1:]):
        assert getattr(cls, f).offset == off, f


def _args(**kw):
    a = _lib.FgAdapterArgs()
    a.hidden = a.weight = a.down = a.up = a.scales = a.adapters = a.out = 256
    a.workspace, a.workspace_bytes = 256, 1 << 20
    a.dtype, a.out_dtype = _lib.FG_DTYPE_BF16, _lib.FG_DTYPE_F32
    a.batch, a.dim, a.vocab, a.rank, a.slots = 0, 60, 100, 16, 3
    a.hidden_stride, a.weight_stride, a.down_stride, a.out_stride = 60, 64, 64, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("bad", [
    dict(hidden=None), dict(weight=None), dict(out=None), dict(down=None), dict(up=None), dict(scales=None),
    dict(dtype=_lib.FG_DTYPE_F32), dict(out_dtype=_lib.FG_DTYPE_F16), dict(batch=-1), dict(dim=0), dict(vocab=0),
    dict(rank=0), dict(rank=4), dict(rank=20), dict(rank=136), dict(slots=-1), dict(reserved=1),
    dict(hidden_stride=59), dict(weight_stride=60), dict(weight_stride=56), dict(down_stride=56),
    dict(down_stride=60), dict(out_stride=99), dict(weight=264), dict(down=264), dict(up=264), dict(hidden=257),
    dict(out=258), dict(workspace=None), dict(workspace=128), dict(workspace_bytes=255)])
def test_refusals(bad):
    lib = _lib.load()
    assert lib.fg_adapter_logits(None, None) == _lib.FG_EINVAL
    assert lib.fg_adapter_logits(_args(), None) == _lib.FG_OK           # empty batch: nothing to do
    assert lib.fg_adapter_logits(_args(**bad), None) == _lib.FG_EINVAL


def test_limits():
    lib = _lib.load()
    for big in (dict(batch=(1 << 20) + 1), dict(dim=(1 << 20) + 8, hidden_stride=1 << 21, weight_stride=1 << 21,
                                                down_stride=1 << 21), dict(vocab=(1 << 28) + 1, out_stride=1 << 29)):
        assert lib.fg_adapter_logits(_args(**big), None) == _lib.FG_ENOTSUP


def test_workspace_size():
    f = _lib.load().fg_adapter_workspace_size
    assert f(64, 4096, 16, 8) >= 64 * 16 * 4
    assert f(64, 4096, 16, 0) > 0 and f(0, 4096, 16, 3) > 0
    assert f(64, 4096, 20, 1) == 0 and f(-1, 4096, 16, 1) == 0 and f(1, 0, 16, 1) == 0


def test_cpu_weight_is_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        AdapterHead(torch.zeros(8, 8, dtype=torch.bfloat16))
