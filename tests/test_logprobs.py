"""Token log probabilities: the argument checks of the C ABI and of the Python
functions that need no GPU, and the structs' layouts."""
import ctypes
import os
import subprocess

import pytest
import torch

from flashgen_b200 import _lib
from flashgen_b200.sampling.logprobs import token_logprobs

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("struct", ["FgLogprobArgs", "FgLogprobGradArgs"])
def test_struct_layout_matches_header(tmp_path, struct):
    cls = getattr(_lib, struct)
    fields = [f[0] for f in cls._fields_]
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flashgen_sampler.h"\nint main(void){\n'
    prog += f'printf("%zu\\n", sizeof({struct}));\n'
    for f in fields:
        prog += f'printf("%zu\\n", offsetof({struct}, {f}));\n'
    c = tmp_path / "probe.c"
    c.write_text(prog + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)])
    vals = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert vals[0] == ctypes.sizeof(cls)
    for f, off in zip(fields, vals[1:]):
        assert getattr(cls, f).offset == off, f


def _args(cls, **kw):
    a = cls()
    a.logits, a.dtype, a.batch, a.vocab, a.row_stride = 16, _lib.FG_DTYPE_F32, 0, 8, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(dtype=7), dict(batch=-1), dict(vocab=0),
                                 dict(row_stride=7), dict(logits=18), dict(top=33), dict(top=-1)])
def test_forward_refusals(bad):
    lib = _lib.load()
    assert lib.fg_token_logprobs(None, None) == _lib.FG_EINVAL
    assert lib.fg_token_logprobs(_args(_lib.FgLogprobArgs), None) == _lib.FG_OK        # empty batch
    assert lib.fg_token_logprobs(_args(_lib.FgLogprobArgs, **bad), None) == _lib.FG_EINVAL


def test_forward_limits():
    lib = _lib.load()
    assert lib.fg_token_logprobs(_args(_lib.FgLogprobArgs, batch=(1 << 30) + 1), None) == _lib.FG_ENOTSUP
    big = (1 << 28) + 1
    assert lib.fg_token_logprobs(_args(_lib.FgLogprobArgs, vocab=big, row_stride=big), None) == _lib.FG_ENOTSUP


@pytest.mark.parametrize("bad", [dict(logits=None), dict(out_grad=None), dict(grad_stride=7), dict(max=None),
                                 dict(logsum=None), dict(grad_entropy=16), dict(reserved=1), dict(out_grad=18),
                                 dict(out_grad=16, grad_stride=9)])
def test_gradient_refusals(bad):
    lib = _lib.load()
    good = dict(max=16, logsum=16, out_grad=32, grad_stride=8)
    assert lib.fg_token_logprobs_grad(None, None) == _lib.FG_EINVAL
    assert lib.fg_token_logprobs_grad(_args(_lib.FgLogprobGradArgs, **good), None) == _lib.FG_OK
    assert lib.fg_token_logprobs_grad(_args(_lib.FgLogprobGradArgs, **{**good, **bad}), None) == _lib.FG_EINVAL


def test_cpu_logits_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        token_logprobs(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64))
