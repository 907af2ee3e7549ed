"""Temperatures at which a quotient leaves the numbers: x / T is an infinity there, not NaN."""
import numpy as np
import pytest
import torch

from flashgen_b200 import Sampler, SamplingParams, _lib
from test_min_p_gpu import BF16, F16, F32, call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("temperature", [1e-37, 1e-38, 1e-45])
@pytest.mark.parametrize("shape", [(1, 40), (3, 5000), (200, 700)])
@pytest.mark.parametrize("min_p,top_k", [(0.1, 0), (0.0, 1), (0.0, 3), (0.0, 0)])
def test_tiny_temperatures(cuda_device, dtype, temperature, shape, min_p, top_k):
    n, v = shape
    rng = np.random.default_rng(v)
    x = -torch.from_numpy(rng.uniform(40, 60, (n, v)).astype(np.float32)).to("cuda", dtype)
    p = {"min_p": np.full(n, min_p, np.float32), "temperature": np.full(n, temperature, np.float32),
         "top_k": np.full(n, top_k), "top_p": np.ones(n, np.float32), "greedy": np.zeros(n, bool)}
    u = np.full(n, 0.5, np.float32)
    # all of a row below 0: -inf everywhere
    r = call(x, u, p)
    assert (r.status.cpu().numpy() & _lib.FG_ROW_ERROR_MASK == _lib.FG_ROW_ALL_MASKED).all()
    assert (r.ids == -1).all() and r.logprobs.isnan().all() and (r.kept == 0).all()
    # a 0 stays one, and is all there is
    x[:, v // 3] = 0.0
    r = call(x, u, p)
    assert (r.ids == v // 3).all() and (r.kept == 1).all() and (r.logprobs == 0).all()
    # the same through fg_sample
    if min_p == 0.0:
        ids = Sampler().sample(x, [SamplingParams(temperature=temperature, top_k=top_k)] * n,
                               uniforms=torch.from_numpy(u).cuda())
        assert (ids == v // 3).all()
    x[:, v // 3] = 60.0
    r = call(x, u, p)
    assert (r.status.cpu().numpy() & _lib.FG_ROW_ERROR_MASK == _lib.FG_ROW_POS_INF).all() and (r.ids == -1).all()
