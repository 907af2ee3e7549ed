"""The PyBind11 module's min-p, linear and clipping entries: argument checks without a GPU,
and one call each on one."""
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
    with pytest.raises(RuntimeError, match="fg_sample_min_p failed: invalid argument"):
        C.sample_min_p(0, C.DTYPE_F32, 2, 10, uniforms=16, out_ids=16, workspace=16, workspace_bytes=100)
    with pytest.raises(RuntimeError, match="fg_linear failed: invalid argument"):
        C.linear(256, 256, 256, C.DTYPE_F32, 2, 8, 8)
    with pytest.raises(RuntimeError, match="fg_linear_grad failed: invalid argument"):
        C.linear_grad(256, 256, 256, C.DTYPE_F16, 2, 8, 8, activation=9)
    with pytest.raises(RuntimeError, match="fg_clip_grad_norm failed: invalid argument"):
        C.clip_grad_norm([(256, 512, 4, C.DTYPE_F32, 9)], 1.0, out_norm=16, workspace=16, workspace_bytes=1 << 20)
    assert C.SamplingParams().min_p == 0.0


def test_workspace_sizes_match_c_abi(C):
    lib = _lib.load()
    assert C.sample_min_p_workspace_size(7, 32000, 100) == lib.fg_sample_min_p_workspace_size(7, 32000, 100) > 0
    assert C.clip_workspace_size(200) == lib.fg_clip_workspace_size(200) > 0


@pytest.mark.gpu
def test_calls(C, cuda_device):
    from flashgen_b200 import clip_grad_norm, fused_linear, sample_min_p
    g = torch.Generator().manual_seed(0)
    st = torch.cuda.current_stream().cuda_stream
    x = torch.randn(5, 64, generator=g).to(torch.bfloat16).cuda()
    w = torch.randn(48, 64, generator=g).to(torch.bfloat16).cuda()
    b = torch.randn(48, generator=g).to(torch.bfloat16).cuda()
    gy = torch.randn(5, 48, generator=g).to(torch.bfloat16).cuda()
    out, z = torch.empty_like(gy), torch.empty(5, 48, device="cuda")
    C.linear(x.data_ptr(), w.data_ptr(), out.data_ptr(), C.DTYPE_BF16, 5, 64, 48, C.ACT_SILU, bias=b.data_ptr(),
             preact=z.data_ptr(), stream=st)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = fused_linear(*leaves, activation="silu")
    assert torch.equal(out, want.detach())
    grads = [torch.empty_like(t) for t in (x, w, b)]
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    C.linear_grad(gy.data_ptr(), x.data_ptr(), w.data_ptr(), C.DTYPE_BF16, 5, 64, 48, C.ACT_SILU, preact=z.data_ptr(),
                  grad_x=grads[0].data_ptr(), grad_weight=grads[1].data_ptr(), grad_bias=grads[2].data_ptr(),
                  workspace=ws.data_ptr(), workspace_bytes=ws.numel(), stream=st)
    assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(want, leaves, gy)))
    clipped, norm = [torch.empty_like(t) for t in grads], torch.empty(1, device="cuda")
    C.clip_grad_norm([(a.data_ptr(), c.data_ptr(), a.numel(), C.DTYPE_BF16, C.DTYPE_BF16)
                      for a, c in zip(grads, clipped)], 0.5, out_norm=norm.data_ptr(), workspace=ws.data_ptr(),
                     workspace_bytes=ws.numel(), stream=st)
    assert float(norm) == float(clip_grad_norm(grads, 0.5)) and all(torch.equal(a, c) for a, c in zip(grads, clipped))
    logits = torch.randn(5, 300, generator=g).cuda()
    u, mp = torch.rand(5, generator=g).cuda(), torch.full((5,), 0.1, device="cuda")
    ids, lp = torch.empty(5, dtype=torch.int64, device="cuda"), torch.empty(5, device="cuda")
    C.sample_min_p(logits.data_ptr(), C.DTYPE_F32, 5, 300, min_p=mp.data_ptr(), uniforms=u.data_ptr(),
                   out_ids=ids.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                   out_logprobs=lp.data_ptr(), stream=st)
    r = sample_min_p(logits, u, mp)
    assert torch.equal(ids, r.ids) and torch.equal(lp, r.logprobs)
