"""A batch of rows with min-p and rows without: what the others ask for changes nothing of a row's
result, and what fg_sample draws without min-p it draws beside it."""
import ctypes

import numpy as np
import pytest
import torch

from flashgen_b200 import Sampler, SamplingParams, _lib, sample_min_p
from flashgen_b200.sampling.decode import DecodeBatch
from flashgen_b200.sampling.host import HostBatchSampler
from flashgen_b200.sampling.sampler import PackedParams
from flashgen_b200.workloads import make_workload
from test_min_p import args

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def test_packed():
    P = SamplingParams
    assert PackedParams.from_params([P(), P(greedy=True)], "cpu").without_min_p is None
    assert PackedParams.from_params([P(min_p=0.1)] * 2, "cpu").without_min_p is None
    p = PackedParams.from_params([P(), P(min_p=0.1), P(greedy=True), P(min_p=0.2, greedy=True)], "cpu")
    assert p.without_min_p.tolist() == [0, 1, 1, 1] and p.greedy.tolist() == [0, 0, 1, 1]
    # what is 0 in 32 bits is no min-p
    p = PackedParams.from_params([P(min_p=1e-60), P(min_p=0.1)], "cpu")
    assert p.min_p.tolist() == [0.0, np.float32(0.1)] and p.without_min_p.tolist() == [0, 1]
    assert PackedParams.from_params([P(min_p=1e-60)], "cpu").min_p is None


def test_refusals():
    lib = _lib.load()
    assert lib.fg_sample_min_p_rows(None, None) == _lib.FG_EINVAL
    assert lib.fg_sample_min_p_rows(ctypes.byref(args()), None) == _lib.FG_EINVAL            # no min_p
    a = args(batch=0)
    a.min_p = 1 << 20
    assert lib.fg_sample_min_p_rows(ctypes.byref(a), None) == _lib.FG_OK
    a.sample.uniforms = None
    assert lib.fg_sample_min_p_rows(ctypes.byref(a), None) == _lib.FG_EINVAL


def workload(n):
    w = make_workload(3, batch=n, seed=3)
    p = w.params
    params = [dict(temperature=float(p.temperature[i]), top_p=float(p.top_p[i]), top_k=int(p.top_k[i]),
                   repetition_penalty=float(p.repetition_penalty[i]), presence_penalty=float(p.presence_penalty[i]),
                   frequency_penalty=float(p.frequency_penalty[i]), greedy=bool(p.greedy[i])) for i in range(n)]
    return w, params


# one row a cluster, and the batch kernel
@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("probs", [False, True])
def test_rows_without_min_p(cuda_device, n, probs):
    w, params = workload(n)
    logits, u, h = w.logits.cuda(), torch.from_numpy(w.uniforms).cuda(), w.histories()
    s = Sampler()

    def draw(min_p):
        ids = s.sample(logits, [SamplingParams(min_p=m, **p) for m, p in zip(min_p, params)], token_histories=h,
                       uniforms=u, return_probs=probs)
        return ids, s.last_status, s.last_probs

    want = draw([0.0] * n)
    all_of_them = draw([0.1] * n)
    for has in ([i == 0 for i in range(n)], [i == n - 1 for i in range(n)], [i % 3 == 1 for i in range(n)],
                [i != 2 for i in range(n)]):
        got = draw([0.1 if k else 0.0 for k in has])
        k = torch.tensor(has, device="cuda")
        for g, a, b in zip(got, want, all_of_them):
            if g is not None:
                assert torch.equal(g[~k], a[~k]) and torch.equal(g[k], b[k])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [700, 60001, 400003])
def test_rows_are_left_as_they_are(cuda_device, dtype, v):
    # NaN, lowest values and bad parameters in the rows that are not gone through
    n = 12
    x = torch.randn(n, v, device="cuda").to(dtype)
    has = torch.arange(n, device="cuda") % 3 == 0
    mp = torch.where(has, 0.1, 0.0)
    mp[1], mp[3] = -0.0, float("nan")
    x[2, 5], x[4] = float("nan"), torch.finfo(dtype).min
    t = torch.full((n,), 0.7, device="cuda")
    t[5] = -1.0
    u = torch.rand(n, device="cuda")
    want = sample_min_p(x, u, mp, temperature=t)
    ids = torch.full((n,), -77, device="cuda")
    status, kept = (torch.full((n,), 99, dtype=torch.int32, device="cuda") for _ in range(2))
    lps, ws = torch.full((n,), 3.5, device="cuda"), torch.zeros(4096, dtype=torch.uint8, device="cuda")
    a = _lib.FgMinPArgs(_lib.FgSampleArgs(
        logits=x.data_ptr(), dtype={F32: 0, F16: 1, BF16: 2}[dtype], batch=n, vocab=v, row_stride=v,
        temperature=t.data_ptr(), uniforms=u.data_ptr(), out_ids=ids.data_ptr(), out_status=status.data_ptr(),
        workspace=ws.data_ptr(), workspace_bytes=ws.numel()), mp.data_ptr(), lps.data_ptr(), kept.data_ptr())
    assert _lib.load().fg_sample_min_p_rows(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == _lib.FG_OK
    assert torch.equal(ids[has], want.ids[has]) and torch.equal(kept[has], want.kept[has])
    assert torch.equal(status[has], want.status[has]) and int(status[3]) & _lib.FG_ROW_BAD_PARAM
    assert torch.equal(lps[has].nan_to_num(9), want.logprobs[has].nan_to_num(9))
    assert (ids[~has] == -77).all() and (status[~has] == 99).all() and (kept[~has] == 99).all() and (lps[~has] == 3.5).all()


@pytest.mark.gpu
def test_decode_and_host_buffers(cuda_device):
    n = 20
    w, params = workload(n)
    logits, u = w.logits.cuda(), torch.from_numpy(w.uniforms).cuda()
    got = []
    for mp in (0.0, 0.1):
        dec = DecodeBatch([SamplingParams(min_p=mp if i == 3 else 0.0, **p) for i, p in enumerate(params)], w.vocab, capacity=64)
        for i, h in enumerate(w.histories()):
            dec.set_history(i, h[:40])
        got.append(torch.stack([dec.step(logits, uniforms=u.roll(k)).clone() for k in range(4)]))
    others = [i for i in range(n) if i != 3]
    assert torch.equal(got[0][:, others], got[1][:, others])
    host = HostBatchSampler(n, w.vocab, w.logits.dtype, w.hist_ids.size, "cuda")
    res = []
    for mp in (None, 0.1, 1.0):
        w.params.min_p = None if mp is None else np.where(np.arange(n) == 3, np.float32(mp), 0)
        res.append(host.sample(w.logits.pin_memory(), w.params, torch.from_numpy(w.hist_ids).pin_memory(),
                               torch.from_numpy(w.hist_offsets).pin_memory(), w.uniforms, w.hist_max_len))
        torch.cuda.synchronize()
        res[-1] = res[-1].clone()
    assert torch.equal(res[0][others], res[1][others]) and torch.equal(res[0][others], res[2][others])
    # min-p of 1 leaves the likeliest token (and its ties)
    want = sample_min_p(logits[3:4], u[3:4], torch.ones(1, device="cuda"), temperature=torch.tensor([w.params.temperature[3]], device="cuda"),
                        greedy=torch.tensor([bool(w.params.greedy[3])], device="cuda"),
                        repetition_penalty=torch.tensor([w.params.repetition_penalty[3]], device="cuda"),
                        presence_penalty=torch.tensor([w.params.presence_penalty[3]], device="cuda"),
                        frequency_penalty=torch.tensor([w.params.frequency_penalty[3]], device="cuda"),
                        history=(torch.tensor(w.histories()[3], dtype=torch.int32, device="cuda"),
                                 torch.tensor([0, len(w.histories()[3])], device="cuda"), len(w.histories()[3])))
    assert int(res[2][3]) == int(want.ids[0])


@pytest.mark.gpu
def test_a_captured_batch_of_both_kinds(cuda_device):
    n, v = 40, 9000
    params = [SamplingParams(min_p=0.1 if i % 4 == 0 else 0.0, temperature=0.8, top_p=0.9) for i in range(n)]
    packed = PackedParams.from_params(params, torch.device("cuda"))
    from flashgen_b200.sampling.sampler import fused_sample
    logits, u = torch.randn(n, v, device="cuda"), torch.rand(n, device="cuda")
    ws = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    out, status = torch.empty(n, dtype=torch.int64, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    fused_sample(logits, packed, u, out=out, status=status, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fused_sample(logits, packed, u, out=out, status=status, workspace=ws)
    for _ in range(2):
        logits.copy_(torch.randn(n, v, device="cuda"))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, fused_sample(logits, packed, u))
