"""Min-p sampling of rows whose finite logits the temperature takes to -inf: such a row has no
token to draw (status, id -1), and nothing of the call before is left in its results."""
import numpy as np
import pytest
import torch

from flashgen_b200 import SamplingParams, _lib, sample_min_p
from flashgen_b200.sampling.decode import DecodeBatch
from test_min_p_gpu import call, check

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (2, 1000), (3, 4096), (2, 4097), (1, 30000), (200, 700)])
@pytest.mark.parametrize("min_p,top_k", [(0.1, 0), (1.0, 0), (0.0, 50), (0.0, 0), (0.2, 7)])
def test_rows_of_the_lowest_value(cuda_device, dtype, shape, min_p, top_k):
    n, v = shape
    x = torch.full(shape, torch.finfo(dtype).min, dtype=dtype, device="cuda")
    p = {"min_p": np.full(n, min_p, np.float32), "temperature": np.full(n, 0.5, np.float32),
         "top_k": np.full(n, top_k), "top_p": np.full(n, 0.9, np.float32), "greedy": np.zeros(n, bool)}
    u = np.linspace(0, 0.99, n, dtype=np.float32)
    warm = {**p, "temperature": np.ones(n, np.float32)}
    # (a call that leaves valid results where the next one's are allocated)
    for q in (warm, p, warm):
        r = call(x, u, q)
        if q is warm:
            check(r, x, u, q)
            assert (r.ids >= 0).all()
        else:
            assert (r.status.cpu().numpy() & _lib.FG_ROW_ERROR_MASK == _lib.FG_ROW_ALL_MASKED).all()
            assert (r.ids == -1).all() and r.logprobs.isnan().all() and (r.kept == 0).all()
        del r
    # one token that stays finite is the only one
    x[:, v // 2] = 0.0
    r = call(x, u, p)
    assert (r.ids == v // 2).all() and (r.kept == 1).all() and (r.logprobs == 0).all()
    # greedy rows do not divide
    x[:, v // 2] = torch.finfo(dtype).min
    r = call(x, u, {**p, "greedy": np.ones(n, bool)})
    assert (r.ids == 0).all() and (r.kept == 1).all()


def test_a_decode_step_keeps_nothing_of_the_one_before(cuda_device):
    dec = DecodeBatch([SamplingParams(min_p=0.1, temperature=0.5)] * 3, vocab=500, capacity=8)
    x = torch.randn(3, 500, device="cuda")
    assert (dec.step(x) >= 0).all()
    x[1] = torch.finfo(F32).min
    assert (dec.step(x) >= 0).tolist() == [True, False, True]
    assert [len(h) for h in dec.histories()] == [2, 1, 2]
    strict = DecodeBatch([SamplingParams(min_p=0.1, temperature=0.5)] * 3, vocab=500, capacity=8, check_errors=True)
    with pytest.raises(RuntimeError, match="all -inf"):
        strict.step(x)


def test_the_positive_side(cuda_device):
    x = torch.full((2, 900), torch.finfo(F32).max, device="cuda")
    t = torch.tensor([0.5, 1.0], device="cuda")
    r = sample_min_p(x, torch.full((2,), 0.5, device="cuda"), torch.full((2,), 0.1, device="cuda"), temperature=t)
    assert (r.status.cpu().numpy() & _lib.FG_ROW_ERROR_MASK).tolist() == [_lib.FG_ROW_POS_INF, 0]
    assert r.ids.tolist() == [-1, 450] and r.kept.tolist() == [0, 900]
