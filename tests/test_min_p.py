"""Min-p sampling without a GPU: parameters, refusals, the reference itself."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from flashgen_b200 import SamplingParams, _lib, sample_min_p
from flashgen_b200.sampling.sampler import PackedParams
from flashgen_b200.sampling.sharded import local_candidates
from min_p_reference import sample_row
from test_abi import HEADER


def test_parameters():
    assert SamplingParams().min_p == 0.0
    SamplingParams(min_p=1.0)
    for bad in (-0.1, 1.1):
        with pytest.raises(ValueError, match="min_p"):
            SamplingParams(min_p=bad)
    p = [SamplingParams(), SamplingParams(min_p=0.25)]
    assert PackedParams.from_params(p[:1], "cpu").min_p is None
    assert PackedParams.from_params(p, "cpu").min_p.tolist() == [0.0, 0.25]


def test_a_shard_is_refused():
    packed = PackedParams.from_params([SamplingParams(min_p=0.1)], "cpu")
    with pytest.raises(ValueError, match="whole row's maximum"):
        local_candidates(torch.zeros(1, 8), packed, torch.zeros(1), None, 0, 16, 4)


def test_python_refusals():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(ValueError, match="logits must be"):
        sample_min_p(x[0], u, u)
    with pytest.raises(ValueError, match="logits must be"):
        sample_min_p(x[:, :0], u, u)
    with pytest.raises(RuntimeError, match="GPU only"):
        sample_min_p(x, u, u)


def args(**kw):
    s = dict(logits=1 << 20, dtype=0, batch=3, vocab=100, hist_max_len=10, row_stride=100, vocab_offset=0,
             vocab_total=0, hist_ids=1 << 16, hist_offsets=1 << 17, temperature=None, top_p=None, top_k=None,
             repetition_penalty=1 << 18, presence_penalty=None, frequency_penalty=None, greedy=None,
             uniforms=1 << 19, out_ids=1 << 21, out_status=None, out_probs=None, workspace=1 << 22,
             workspace_bytes=1 << 20)
    s.update(kw)
    return _lib.FgMinPArgs(_lib.FgSampleArgs(**s), None, None, None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(logits=(1 << 20) + 2), dict(dtype=3), dict(batch=-1), dict(vocab=0), dict(row_stride=99),
    dict(uniforms=None), dict(out_ids=None), dict(hist_ids=None), dict(hist_offsets=None), dict(hist_max_len=-1),
    dict(vocab_offset=5), dict(vocab_offset=-1), dict(vocab_total=200), dict(workspace=None),
    dict(workspace=(1 << 22) + 4), dict(workspace_bytes=100),
])
def test_c_refusals(bad):
    assert _lib.load().fg_sample_min_p(ctypes.byref(args(**bad)), None) == _lib.FG_EINVAL


def test_c_limits_and_workspace():
    lib = _lib.load()
    assert lib.fg_sample_min_p(None, None) == _lib.FG_EINVAL
    assert lib.fg_sample_min_p(ctypes.byref(args(batch=0)), None) == _lib.FG_OK
    assert lib.fg_sample_min_p(ctypes.byref(args(batch=(1 << 24) + 1)), None) == _lib.FG_ENOTSUP
    assert lib.fg_sample_min_p(ctypes.byref(args(vocab=(1 << 28) + 1, row_stride=1 << 29)), None) == _lib.FG_ENOTSUP
    size = lib.fg_sample_min_p_workspace_size
    assert size(5, 100, 0) == 8 and size(0, 100, 0) == 8
    assert size(5, 100, 10) > size(5, 100, 0) and size(5, 100000, 40000) > size(5, 100000, 10)
    assert size(5, 100, 10) == size(5, 100, 32)
    assert size(-1, 100, 0) == size(5, 0, 0) == size(5, 100, -1) == 0


def test_struct_layout(tmp_path):
    fields = [f for f, *_ in _lib.FgMinPArgs._fields_]
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flashgen_sampler.h"\nint main(void){\n'
    prog += 'printf("%zu\\n", sizeof(FgMinPArgs));\n' + "".join(
        f'printf("%zu\\n", offsetof(FgMinPArgs, {f}));\n' for f in fields)
    c = tmp_path / "probe.c"
    c.write_text(prog + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.dirname(HEADER), str(c), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert got == [ctypes.sizeof(_lib.FgMinPArgs)] + [getattr(_lib.FgMinPArgs, f).offset for f in fields]


def test_the_reference():
    x = np.log(np.array([0.1, 0.4, 0.3, 0.2], dtype=np.float64)).astype(np.float32)
    assert sample_row(x, 0.0, 0.0).id == 1 and sample_row(x, 0.95, 0.0).id == 0
    r = sample_row(x, 0.5, 0.6)                         # 0.4 and 0.3 are left: 4/7, 3/7
    assert (r.id, r.kept) == (1, 2) and abs(np.exp(r.logprob) - 4 / 7) < 1e-6
    assert sample_row(x, 0.58, 0.6).id == 2
    assert sample_row(x, 0.99, 0.3, top_k=2).id == 2 and sample_row(x, 0.99, 0.3, top_k=2).kept == 2
    assert sample_row(x, 0.99, 0.3, top_p=0.4).kept == 1          # of 4/9: the next begins at 0.444
    assert sample_row(x, 0.99, 0.3, top_p=0.5).kept == 2
    assert sample_row(np.zeros(5), 0.5, 1.0).id == 2 and sample_row(np.zeros(5), 0.5, 1.0).kept == 5
    assert sample_row(x, 0.5, 0.1, greedy=True).id == 1
    assert sample_row(x, 0.0, 0.1, rep=2.0, history=[1, 1]).id == 2       # log 0.4 doubled is below log 0.3
