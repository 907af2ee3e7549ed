"""Min-p sampling at the sizes where its kernels change their way: as many candidates as a
row has room for and one more (in one CTA and in a cluster), a bin of as many tokens as are put
in order and one more, top-k and histories at the first kernel's limits, and long rows with
penalties whose keys are worked out anew in every pass."""
import numpy as np
import pytest
import torch

from test_min_p_gpu import BF16, F16, F32, call, check, draw_params, rows

pytestmark = pytest.mark.gpu


def plain(n, **kw):
    p = {"min_p": np.full(n, 0.2, np.float32), "temperature": np.ones(n, np.float32), "top_k": np.zeros(n, int),
         "top_p": np.ones(n, np.float32), "greedy": np.zeros(n, bool)}
    return {k: np.full(n, kw[k], p[k].dtype) if k in kw else a for k, a in p.items()}


# 600 rows take one CTA each, two rows a cluster each; 4200 words are one CTA's however few rows
@pytest.mark.parametrize("batch,v", [(600, 12000), (2, 30000), (2, 200000), (3, 4200)])
@pytest.mark.parametrize("count", [4095, 4096, 4097])
def test_candidates(cuda_device, batch, v, count):
    rng = np.random.default_rng(count)
    x = torch.full((batch, v), -20.0, device="cuda")
    at = torch.from_numpy(rng.permutation(v)[:count]).cuda()
    x[:, at] = torch.from_numpy(rng.random((batch, count)).astype(np.float32)).cuda()
    u = rng.random(batch, dtype=np.float32)
    for kw in ({}, {"top_p": 0.7}, {"top_k": 300}):
        p = plain(batch, **kw)
        r = call(x, u, p)
        check(r, x, u, p, rows=range(0, batch, max(1, batch // 6)))
        if not kw:
            assert (r.kept == count).all()


# candidates of a single slice of a cluster's, in ascending order: all are new maxima
@pytest.mark.parametrize("count", [4095, 4096, 4097, 12000])
def test_candidates_of_one_slice(cuda_device, count):
    x = torch.full((1, 200000), -20.0, device="cuda")
    x[0, :count] = torch.linspace(0, 1, count, device="cuda")
    for src in (x, x.flip(1)):
        p, u = plain(1), np.array([0.37], np.float32)
        r = call(src, u, p)
        check(r, src, u, p)
        assert int(r.kept) == count


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("ties", [64, 65, 1023, 1024, 1025])
@pytest.mark.parametrize("batch", [2, 500])
def test_ties_in_one_bin(cuda_device, dtype, ties, batch):
    # among distinct values, below and above them
    rng = np.random.default_rng(ties)
    v = 9000
    x = torch.full((batch, v), -30.0)
    at = rng.permutation(v)
    x[:, at[:ties]] = 0.5
    x[:, at[ties:ties + 200]] = torch.from_numpy(rng.random((batch, 200)).astype(np.float32)) * 0.4 + 0.55
    x[:, at[ties + 200:ties + 400]] = torch.from_numpy(rng.random((batch, 200)).astype(np.float32)) * 0.4 + 0.05
    x = x.to("cuda", dtype)
    u = rng.random(batch, dtype=np.float32)
    for kw in ({}, {"top_k": 210}, {"top_p": 0.5}, {"top_k": 200 + ties + 3, "top_p": 0.9}, {"min_p": 0.0}):
        p = plain(batch, **kw)
        check(call(x, u, p), x, u, p, rows=range(0, batch, max(1, batch // 4)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top_k", [1, 511, 512, 513])
@pytest.mark.parametrize("shape", [(3, 513), (3, 5000), (1, 100000), (450, 2000)])
def test_top_k_without_min_p(cuda_device, dtype, top_k, shape):
    rng = np.random.default_rng(top_k)
    n, v = shape
    x, u = rows(n, v, dtype, rng), rng.random(n, dtype=np.float32)
    p = plain(n, min_p=0.0, top_k=top_k, top_p=0.95)
    check(call(x, u, p), x, u, p, rows=range(0, n, max(1, n // 6)))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("length", [2048, 2049, 4095, 4096, 4097])
def test_history_lengths(cuda_device, dtype, length):
    rng = np.random.default_rng(length)
    n, v = 5, 9000
    x, u = rows(n, v, dtype, rng), rng.random(n, dtype=np.float32)
    history = [rng.permutation(v)[:length], rng.integers(0, v, length), rng.integers(0, 3, length), [], [5]]
    pen = {"rep": np.full(n, 1.3, np.float32), "freq": np.full(n, 0.2, np.float32)}
    for p in (plain(n), plain(n, top_k=40, min_p=0.0), draw_params(n, rng)):
        check(call(x, u, p, pen, history), x, u, p, pen, history)


# rows of which a cluster of eight holds no cache of keys
@pytest.mark.parametrize("dtype,v", [(F32, 300001), (BF16, 400003), (F16, 333333)])
@pytest.mark.parametrize("length", [9, 3000, 20000])
def test_long_rows_with_penalties(cuda_device, dtype, v, length):
    rng = np.random.default_rng(v + length)
    n = 3
    x, u = rows(n, v, dtype, rng), rng.random(n, dtype=np.float32)
    best = x.float().argmax(1).cpu().numpy()
    history = [np.concatenate([rng.integers(0, v, length), [best[i]] * i]) for i in range(n)]
    pen = {"rep": np.array([1.2, 1.0, 0.9], np.float32), "pres": np.full(n, 0.4, np.float32),
           "freq": np.array([0.0, 0.3, 0.5], np.float32)}
    for kw in ({"min_p": 0.0}, {"min_p": 0.0, "top_p": 0.8}, {"min_p": 0.0, "top_k": 1000}, {"min_p": 0.05}):
        p = plain(n, temperature=0.8, **kw)
        check(call(x, u, p, pen, history), x, u, p, pen, history)
    # greedy rows, and rows that the whole row's pass alone can tell
    p = plain(n, min_p=0.0, greedy=True)
    check(call(x, u, p, pen, history), x, u, p, pen, history)
