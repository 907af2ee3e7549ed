"""Rows of fg_sample whose finite logits the temperature takes to an infinity: they are reported, and
beside rows with min-p the same as without."""
import pytest
import torch

from flashgen_b200 import Sampler, SamplingParams, _lib

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# one row a cluster, and the batch kernel
@pytest.mark.parametrize("batch", [1, 4, 400])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [1, 7, 1000, 20001])
@pytest.mark.parametrize("kw", [{}, {"top_k": 5}, {"top_p": 0.9}, {"top_k": 40, "top_p": 0.8}])
@pytest.mark.parametrize("history", [False, True])
def test_quotients_that_leave_the_numbers(cuda_device, batch, dtype, v, kw, history):
    x = torch.zeros(batch, v, device="cuda").to(dtype)
    x[::2] = torch.finfo(dtype).min
    x[1::4] = torch.finfo(dtype).max
    u = torch.rand(batch, device="cuda")
    s = Sampler(check_errors=False)
    h = [[0, 0]] * batch if history else None
    for min_p in (0.0, 0.2, None):
        params = [SamplingParams(temperature=0.5, repetition_penalty=1.1 if history else 1.0,
                                 min_p=min_p if min_p is not None else 0.1 * (i % 8 >= 4), **kw) for i in range(batch)]
        for probs in (False, True):
            ids = s.sample(x, params, uniforms=u, token_histories=h, return_probs=probs)
            status = s.last_status & _lib.FG_ROW_ERROR_MASK
            assert (ids[::2] == -1).all() and (status[::2] == _lib.FG_ROW_ALL_MASKED).all()
            if v > 1 or not history:              # (the largest logit of one column is penalised to a finite one)
                assert (ids[1::4] == -1).all() and (status[1::4] == _lib.FG_ROW_POS_INF).all()
            assert (ids[3::4] >= 0).all() and (status[3::4] == 0).all()
            if probs:
                assert (s.last_probs[::2] == 0).all() and s.last_probs.isfinite().all()
    # without the temperature they are ordinary rows
    ids = s.sample(x, [SamplingParams(**kw)] * batch, uniforms=u)
    assert (ids >= 0).all() and (s.last_status & _lib.FG_ROW_ERROR_MASK == 0).all()
