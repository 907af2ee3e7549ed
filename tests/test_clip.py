"""Refusals of the gradient norm and clipping, without a GPU."""
import ctypes
import math

import pytest
import torch

from flashgen_b200 import _lib, clip_grad_norm, grad_norm


def test_python_refusals():
    g = torch.ones(4)
    for bad in ([], ()):
        with pytest.raises(ValueError, match="no gradients"):
            clip_grad_norm(bad, 1.0)
        with pytest.raises(ValueError, match="no gradients"):
            grad_norm(bad)
    with pytest.raises(TypeError, match="NoneType"):
        clip_grad_norm([g, None], 1.0)
    with pytest.raises(TypeError, match="float64"):
        grad_norm(g.double())
    with pytest.raises(TypeError, match="sparse"):
        grad_norm(torch.eye(3).to_sparse())
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm(g, bad)
    for bad in (0.0, -2.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            clip_grad_norm(g, 1.0, scale=bad)
        with pytest.raises(ValueError, match="scale"):
            grad_norm(g, scale=bad)
    with pytest.raises(ValueError, match="2 gradients, 1 results"):
        clip_grad_norm([g, g], 1.0, out=[g])
    with pytest.raises(ValueError, match="shapes"):
        clip_grad_norm([g], 1.0, out=[torch.ones(2, 2)])
    with pytest.raises(RuntimeError, match="GPU only"):
        clip_grad_norm([g], 1.0)


def _call(tensors, max_norm=1.0, scale=1.0, count=None, norm=4096, ws=8192, need=1 << 30, reserved=0):
    table = (_lib.FgGradTensor * max(1, len(tensors)))(*[_lib.FgGradTensor(*t) for t in tensors])
    a = _lib.FgClipArgs(ctypes.addressof(table), len(tensors) if count is None else count, reserved, max_norm, scale,
                        norm, ws, need)
    return _lib.load().fg_clip_grad_norm(ctypes.byref(a), None)


@pytest.mark.parametrize("tensors", [
    [(1 << 20, 1 << 21, 100, 7, 0)],                                     # bad type
    [(1 << 20, 1 << 21, 100, 0, 3)],                                     # bad result type
    [(1 << 20, 1 << 21, -1, 0, 0)],                                      # bad count
    [(0, 1 << 21, 100, 0, 0)],                                           # no gradients
    [((1 << 20) + 2, 1 << 21, 100, 0, 0)],                               # gradients not aligned
    [(1 << 20, (1 << 21) + 1, 100, 0, 1)],                               # result not aligned
    [(1 << 20, (1 << 20) + 4, 100, 0, 0)],                               # a part of its own gradients
    [(1 << 20, 1 << 20, 100, 0, 1)],                                     # the same place as another type
    [(1 << 20, 1 << 20, 100, 0, 0), (1 << 20, 1 << 20, 100, 0, 0)],      # a tensor twice
    [(1 << 20, 1 << 22, 100, 0, 0), (1 << 21, (1 << 22) + 396, 100, 0, 0)],   # results that meet
    [(1 << 20, 1 << 22, 100, 0, 0), ((1 << 22) + 396, None, 9, 0, 0)],   # a result over another's gradients
    [((1 << 22) + 396, None, 9, 0, 0), (1 << 20, 1 << 22, 100, 0, 0)],
])
def test_c_refusals(tensors):
    assert _call(tensors) == _lib.FG_EINVAL


def test_c_refusals_of_the_call():
    one = [(1 << 20, 1 << 21, 100, 0, 0)]
    lib = _lib.load()
    assert lib.fg_clip_grad_norm(None, None) == _lib.FG_EINVAL
    for kw in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(scale=0.0), dict(scale=math.inf),
               dict(scale=math.nan), dict(count=-1), dict(norm=None), dict(norm=2), dict(ws=None), dict(ws=4),
               dict(need=lib.fg_clip_workspace_size(1) - 1), dict(reserved=1)):
        assert _call(one, **kw) == _lib.FG_EINVAL, kw
    assert _call(one, count=(1 << 20) + 1) == _lib.FG_ENOTSUP
    assert lib.fg_clip_workspace_size(-1) == 0 and lib.fg_clip_workspace_size((1 << 20) + 1) == 0
    assert 0 < lib.fg_clip_workspace_size(0) < lib.fg_clip_workspace_size(96) < lib.fg_clip_workspace_size(2000)


def test_struct_layout(tmp_path):
    from test_abi import HEADER
    import os
    import subprocess
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flashgen_sampler.h"\nint main(void){\n'
    want = []
    for s in (_lib.FgGradTensor, _lib.FgClipArgs):
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
