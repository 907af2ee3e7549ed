"""Min-p sampling with histories whose longest is given as 0 or too short: the penalties hold, or
the row is marked."""
import ctypes

import numpy as np
import pytest
import torch

from flashgen_b200 import _lib, sample_min_p
from flashgen_b200.sampling.host import HostBatchSampler
from flashgen_b200.workloads import make_workload
from min_p_reference import sample_row
from test_min_p import args

F32 = torch.float32


def test_a_bound_of_0_takes_a_table():
    # (a workspace without one is refused before anything is launched)
    lib = _lib.load()
    size = lib.fg_sample_min_p_workspace_size
    assert lib.fg_sample_min_p(ctypes.byref(args(hist_max_len=0, workspace_bytes=size(3, 100, 1) - 1)), None) == _lib.FG_EINVAL
    assert size(3, 100, 1) > size(3, 100, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [0, 1, 2])
@pytest.mark.parametrize("v,min_p", [(50, 0.2), (5000, 0.2), (300001, 0.0)])
def test_penalties_hold(cuda_device, bound, v, min_p):
    x = torch.zeros(3, v, device="cuda")
    x[:, 7], x[:, 3] = 9.0, 8.0
    ids = torch.tensor([7, 7, 3], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 0, 2, 3], device="cuda")
    r = sample_min_p(x, torch.zeros(3, device="cuda"), torch.full((3,), min_p, device="cuda"),
                     frequency_penalty=torch.full((3,), 4.0, device="cuda"), history=(ids, offsets, bound))
    assert r.ids.tolist() == [7, 3, 7] and (r.status.cpu().numpy() & _lib.FG_ROW_ERROR_MASK == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("v,min_p", [(500, 0.2), (300001, 0.0)])
def test_too_many_ids_are_marked(cuda_device, v, min_p):
    x = torch.zeros(2, v, device="cuda")
    ids = torch.arange(200, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 199, 200], device="cuda")
    r = sample_min_p(x, torch.zeros(2, device="cuda"), torch.full((2,), min_p, device="cuda"),
                     frequency_penalty=torch.ones(2, device="cuda"), history=(ids, offsets, 0))
    assert r.ids[0] == -1 and int(r.status[0]) & _lib.FG_ROW_BAD_PARAM
    assert r.ids[1] == 0 and int(r.status[1]) & _lib.FG_ROW_ERROR_MASK == 0


@pytest.mark.gpu
def test_host_buffers_without_a_bound(cuda_device):
    # up to 15 ids a row, and the call's default bound
    w = make_workload(2, batch=16, seed=2)
    w.params.min_p = np.full(16, 0.1, np.float32)
    history = [h[:i] for i, h in enumerate(w.histories())]
    flat = torch.from_numpy(np.concatenate([np.asarray(h, np.int32) for h in history])).pin_memory()
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum([len(h) for h in history])])).pin_memory()
    host = HostBatchSampler(16, w.vocab, w.logits.dtype, w.hist_ids.size, "cuda")
    ids = host.sample(w.logits.pin_memory(), w.params, flat, offsets, w.uniforms)
    torch.cuda.synchronize()
    x = w.logits.float().numpy()
    for i in range(16):
        want = sample_row(x[i], w.uniforms[i], 0.1, 0.7, 50, 0.95, rep=1.1, pres=0.2, freq=0.1, history=history[i])
        assert want.near or int(ids[i]) == want.id
