"""The PyBind11 module's log-probability and LM-head entries: argument checks
without a GPU, and one call each on one."""
import importlib

import pytest
import torch

from flashgen_b200 import _lib
from flashgen_b200 import build as _build


@pytest.fixture(scope="module")
def C():
    _lib.load()
    _build.build_bindings()
    return importlib.import_module("flashgen_b200._C")


def test_errors_raise(C):
    with pytest.raises(RuntimeError, match="fg_token_logprobs failed: invalid argument"):
        C.token_logprobs(0, C.DTYPE_F32, 2, 10)
    with pytest.raises(RuntimeError, match="fg_token_logprobs_grad failed: invalid argument"):
        C.token_logprobs_grad(16, C.DTYPE_F32, 2, 10, 0, 16, 16)
    with pytest.raises(RuntimeError, match="fg_adapter_logits failed: invalid argument"):
        C.adapter_logits(256, 256, 256, C.DTYPE_F32, C.DTYPE_F32, 2, 64, 10, 256, 1 << 20)


def test_workspace_size_matches_c_abi(C):
    f = _lib.load().fg_adapter_workspace_size
    for b, d, r, s in ((1, 64, 16, 2), (300, 4096, 64, 9), (7, 100, 8, 0)):
        assert C.adapter_workspace_size(b, d, r, s) == f(b, d, r, s) > 0


@pytest.mark.gpu
def test_calls(C, cuda_device):
    from flashgen_b200 import AdapterHead, token_logprobs, token_logprobs_grad
    g = torch.Generator().manual_seed(0)
    st = torch.cuda.current_stream().cuda_stream
    w = torch.randn(300, 64, generator=g).to(torch.bfloat16).cuda()
    h = torch.randn(5, 64, generator=g).to(torch.bfloat16).cuda()
    out = torch.empty(5, 300, device="cuda")
    need = C.adapter_workspace_size(5, 64)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    C.adapter_logits(h.data_ptr(), w.data_ptr(), out.data_ptr(), C.DTYPE_BF16, C.DTYPE_F32, 5, 64, 300,
                     ws.data_ptr(), need, stream=st)
    assert torch.equal(out, AdapterHead(w).logits(h, out_dtype=torch.float32))
    t = torch.arange(5, device="cuda")
    r = token_logprobs(out, t)
    lp = torch.empty(5, device="cuda")
    C.token_logprobs(out.data_ptr(), C.DTYPE_F32, 5, 300, tokens=t.data_ptr(), out_logprobs=lp.data_ptr(), stream=st)
    assert torch.equal(lp, r.logprobs)
    grad, ones = torch.empty_like(out), torch.ones(5, device="cuda")
    C.token_logprobs_grad(out.data_ptr(), C.DTYPE_F32, 5, 300, r.max.data_ptr(), r.logsum.data_ptr(),
                          grad.data_ptr(), tokens=t.data_ptr(), grad_logprobs=ones.data_ptr(), stream=st)
    assert torch.equal(grad, token_logprobs_grad(out, t, r.max, r.logsum, ones))
