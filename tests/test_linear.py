"""Refusals of the fused linear block, without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

from flashgen_b200 import HeadBlock, _lib, fused_linear
from test_abi import HEADER

BF16 = torch.bfloat16


def test_python_refusals():
    x, w = torch.zeros(3, 8, dtype=BF16), torch.zeros(4, 8, dtype=BF16)
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="weight must be"):
        fused_linear(x, w[0])
    with pytest.raises(ValueError, match=r"x must be \[..., 8\]"):
        fused_linear(x[:, :7], w)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        fused_linear(x.float(), w.float())
    with pytest.raises(TypeError, match="x must be"):
        fused_linear(x.half(), w)
    with pytest.raises(TypeError, match="bias must be"):
        fused_linear(x, w, torch.zeros(4))
    with pytest.raises(ValueError, match="bias must be"):
        fused_linear(x, w, torch.zeros(1, dtype=BF16))
    with pytest.raises(ValueError, match="residual must be"):
        fused_linear(x, w, None, torch.zeros(4, dtype=BF16))
    with pytest.raises(RuntimeError, match="GPU only"):
        fused_linear(x, w)
    with pytest.raises(ValueError, match="square"):
        HeadBlock(w)
    with pytest.raises(ValueError, match="activation"):
        HeadBlock(w, residual=False, activation="swish")


def linear_args(**kw):
    a = dict(x=1 << 20, weight=1 << 22, bias=None, residual=None, out=1 << 24, preact=None, workspace=None,
             workspace_bytes=0, dtype=2, tokens=5, inner=64, outer=32, activation=0, reserved=0, x_stride=64,
             weight_stride=64, residual_stride=32, out_stride=32, preact_stride=32)
    a.update(kw)
    return _lib.FgLinearArgs(**a)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(weight=None), dict(out=None), dict(dtype=0), dict(dtype=3), dict(tokens=-1), dict(inner=0),
    dict(outer=0), dict(activation=5), dict(activation=-1), dict(reserved=1), dict(x_stride=63),
    dict(weight_stride=63), dict(out_stride=31), dict(x=(1 << 20) + 1), dict(bias=3), dict(preact=(1 << 25) + 2),
    dict(preact=1 << 25, preact_stride=31), dict(residual=1 << 25, residual_stride=31),
    dict(out=1 << 20), dict(out=(1 << 22) + 2), dict(bias=(1 << 24) + 64), dict(preact=(1 << 24) + 64),
    dict(residual=(1 << 24) + 2), dict(residual=1 << 24, residual_stride=40),       # not quite the result
    dict(x_stride=65),                                                              # needs a workspace
    dict(x_stride=65, workspace=128, workspace_bytes=1 << 20),                      # not aligned
])
def test_c_refusals(bad):
    assert _lib.load().fg_linear(ctypes.byref(linear_args(**bad)), None) == _lib.FG_EINVAL


def test_c_limits_and_workspace():
    lib = _lib.load()
    assert lib.fg_linear(None, None) == _lib.FG_EINVAL
    assert lib.fg_linear(ctypes.byref(linear_args(tokens=0)), None) == _lib.FG_OK
    for over in (dict(tokens=(1 << 20) + 1), dict(inner=(1 << 20) + 8, x_stride=1 << 22, weight_stride=1 << 22)):
        assert lib.fg_linear(ctypes.byref(linear_args(**over)), None) == _lib.FG_ENOTSUP
    size = lambda **kw: lib.fg_linear_workspace_size(ctypes.byref(linear_args(**kw)))  # noqa: E731
    assert size() == 0 and size(dtype=0) == 0
    assert size(x_stride=65) == 768                        # 5 rows of 64, in 256s
    assert size(x=(1 << 20) + 2) == 768 and size(weight_stride=68) == 4096
    assert size(x_stride=65, tokens=1) == 0                # one row has no stride


def grad_args(**kw):
    a = dict(grad_out=1 << 20, x=1 << 21, weight=1 << 22, preact=1 << 23, grad_x=1 << 24, grad_weight=1 << 25,
             grad_bias=1 << 26, workspace=1 << 27, workspace_bytes=1 << 20, dtype=1, tokens=5, inner=64, outer=32,
             activation=4, reserved=0, grad_out_stride=32, x_stride=64, weight_stride=64, preact_stride=32,
             grad_x_stride=64, grad_weight_stride=64)
    a.update(kw)
    return _lib.FgLinearGradArgs(**a)


@pytest.mark.parametrize("bad", [
    dict(grad_out=None), dict(x=None), dict(weight=None), dict(preact=None), dict(dtype=0), dict(tokens=-1),
    dict(activation=5), dict(reserved=7), dict(grad_out_stride=31), dict(x_stride=63), dict(weight_stride=63),
    dict(preact_stride=31), dict(grad_x_stride=63), dict(grad_weight_stride=63), dict(grad_bias=5),
    dict(workspace=None), dict(workspace_bytes=100), dict(grad_x=1 << 21), dict(grad_weight=1 << 22),
    dict(grad_x=1 << 25), dict(grad_bias=(1 << 25) + 2), dict(grad_bias=1 << 20),
])
def test_c_grad_refusals(bad):
    assert _lib.load().fg_linear_grad(ctypes.byref(grad_args(**bad)), None) == _lib.FG_EINVAL


def test_struct_layout(tmp_path):
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flashgen_sampler.h"\nint main(void){\n'
    want = []
    for s in (_lib.FgLinearArgs, _lib.FgLinearGradArgs):
        prog += f'printf("%zu\\n", sizeof({s.__name__}));\n'
        want.append(ctypes.sizeof(s))
        for f, *_ in s._fields_:
            prog += f'printf("%zu\\n", offsetof({s.__name__}, {f}));\n'
            want.append(getattr(s, f).offset)
    c = tmp_path / "probe.c"
    c.write_text(prog + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.dirname(HEADER), str(c), "-o", str(exe)])
    assert [int(v) for v in subprocess.check_output([str(exe)]).split()] == want
