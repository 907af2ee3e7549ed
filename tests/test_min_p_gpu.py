"""Min-p sampling against its 64-bit definition (min_p_reference.py).

Ids and kept counts have to be equal (rows within 1e-9 of a border between two tokens aside:
`near`). Log probabilities: the fp32 rounding of the result (2^-24 of it), the 64-bit terms,
and the masses' rounding to integers, up to V units of 2^-46 in the sum: 2^-24 |lp| + 1e-7."""
import numpy as np
import pytest
import torch

from flashgen_b200 import Sampler, SamplingParams, _lib, sample_min_p
from flashgen_b200.sampling.decode import DecodeBatch
from flashgen_b200.sampling.host import HostBatchSampler
from flashgen_b200.workloads import make_workload
from min_p_reference import sample_row

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def draw_params(n, rng, kinds="mixed"):
    p = {"min_p": rng.choice([0.02, 0.1, 0.5], n), "temperature": rng.uniform(0.4, 1.6, n), "top_k": np.zeros(n, int),
         "top_p": np.ones(n), "greedy": np.zeros(n, bool)}
    if kinds == "mixed":
        p["min_p"] = rng.choice([0.0, 1e-6, 0.001, 0.05, 0.3, 1.0], n)
        p["temperature"] = rng.choice([0.3, 1.0, 0.7, 1.7], n)
        p["top_k"] = rng.choice([-1, 0, 1, 5, 50, 700, 100000], n)
        p["top_p"] = rng.choice([1.0, 0.999, 0.9, 0.5, 0.05], n)
        p["greedy"] = rng.random(n) < 0.1
    p["temperature"] = p["temperature"].astype(np.float32)
    p["min_p"], p["top_p"] = p["min_p"].astype(np.float32), p["top_p"].astype(np.float32)
    return p


def call(logits, u, p, pen=None, history=None, **kw):
    t = lambda a, d: None if a is None else torch.as_tensor(np.asarray(a)).to("cuda", d)  # noqa: E731
    pen = pen or {}
    hist = None
    if history is not None:
        flat = np.concatenate([np.asarray(h, dtype=np.int32) for h in history]) if history else np.zeros(0, np.int32)
        offs = np.concatenate([[0], np.cumsum([len(h) for h in history])])
        hist = (t(flat, torch.int32), t(offs, torch.int64), max(len(h) for h in history))
    return sample_min_p(logits, t(u, F32), t(p["min_p"], F32), temperature=t(p["temperature"], F32),
                        top_k=t(p["top_k"], torch.int32), top_p=t(p["top_p"], F32), greedy=t(p["greedy"], torch.bool),
                        repetition_penalty=t(pen.get("rep"), F32), presence_penalty=t(pen.get("pres"), F32),
                        frequency_penalty=t(pen.get("freq"), F32), history=hist, **kw)


def check(r, logits, u, p, pen=None, history=None, rows=None):
    ids, lps, kept = r.ids.cpu().numpy(), r.logprobs.cpu().numpy(), r.kept.cpu().numpy()
    status = r.status.cpu().numpy()
    x = logits.float().cpu().numpy()
    for i in range(len(ids)) if rows is None else rows:
        want = sample_row(x[i], u[i], p["min_p"][i], p["temperature"][i], p["top_k"][i], p["top_p"][i], p["greedy"][i],
                          **{k: v[i] for k, v in (pen or {}).items()}, history=() if history is None else history[i])
        assert status[i] & _lib.FG_ROW_ERROR_MASK == 0, (i, status[i])
        if want.near:
            continue
        assert (ids[i], kept[i]) == (want.id, want.kept), (i, {k: v[i] for k, v in p.items()})
        assert abs(lps[i] - want.logprob) <= 2.0 ** -24 * abs(want.logprob) + 1e-7, (i, lps[i], want.logprob)


def rows(n, v, dtype, rng, scale=2.5):
    return torch.from_numpy((rng.standard_normal((n, v)) * scale).astype(np.float32)).to("cuda", dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 7), (4, 33), (70, 1000), (9, 4097), (20, 32001), (3, 50257)])
@pytest.mark.parametrize("kinds", ["plain", "mixed"])
def test_against_the_definition(cuda_device, dtype, shape, kinds):
    rng = np.random.default_rng(shape[1])
    n, v = shape
    logits, u, p = rows(n, v, dtype, rng), rng.random(n, dtype=np.float32), draw_params(n, rng, kinds)
    check(call(logits, u, p), logits, u, p)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kinds", ["plain", "mixed"])
def test_long_rows(cuda_device, dtype, kinds):
    for n, v in ((1, 256000), (2, 300001), (40, 128256)):
        rng = np.random.default_rng(v)
        logits, u, p = rows(n, v, dtype, rng), rng.random(n, dtype=np.float32), draw_params(n, rng, kinds)
        check(call(logits, u, p), logits, u, p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_penalties_and_histories(cuda_device, dtype):
    rng = np.random.default_rng(5)
    n, v = 60, 5000
    logits, u, p = rows(n, v, dtype, rng), rng.random(n, dtype=np.float32), draw_params(n, rng)
    history = [rng.integers(0, v if i % 3 else 40, rng.integers(0, 900)) if i % 5 else [] for i in range(n)]
    history[7] = np.arange(v)                               # every column (longer than the kernel's own table)
    best = logits.float().argmax(1).cpu().numpy()
    for i in range(0, n, 4):
        history[i] = np.concatenate([history[i], [best[i]] * (i % 7)])   # the likeliest token is penalised away
    pen = {"rep": rng.choice([1.0, 1.3, 0.8], n).astype(np.float32), "pres": rng.choice([0.0, 0.7], n).astype(np.float32),
           "freq": rng.choice([0.0, 0.4], n).astype(np.float32)}
    check(call(logits, u, p, pen, history), logits, u, p, pen, history)
    for one in ("rep", "pres", "freq"):
        check(call(logits, u, p, {one: pen[one]}, history), logits, u, p, {one: pen[one]}, history)
    # a history that names each id once, longer than any table in shared memory
    one = {k: v_[:1] for k, v_ in p.items()}
    big = rows(1, 60000, dtype, rng)
    h = [rng.permutation(60000)[:50000]]
    check(call(big, u[:1], one, {"freq": pen["freq"][:1] + 1}, h), big, u[:1], one, {"freq": pen["freq"][:1] + 1}, h)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_masks_ties_and_flat_rows(cuda_device, dtype):
    rng = np.random.default_rng(6)
    v = 20011
    low = torch.finfo(dtype).min
    base = rows(12, v, dtype, rng)
    keep = torch.from_numpy(rng.random((12, v)) < 0.003).cuda()
    keep[:, 17] = True
    kinds = [torch.where(keep, base, torch.tensor(-torch.inf, device="cuda", dtype=dtype)),
             torch.where(keep, base, torch.tensor(low, device="cuda", dtype=dtype)),
             torch.zeros_like(base), torch.full_like(base, -3.0),                       # all equal
             torch.where(keep, 4.0, 0.0).to(dtype), (base.float().round()).to(dtype),   # many ties
             torch.where(torch.arange(v, device="cuda") == 9, 50.0, 0.0).to(dtype).expand(12, v),
             -base.abs(), torch.where(base > 0, 0.0, -0.0).to(dtype)]                   # signed zeros are equal
    for k, logits in enumerate(kinds):
        u, p = rng.random(12, dtype=np.float32), draw_params(12, rng)
        check(call(logits, u, p), logits, u, p)
    # one token left
    one = torch.full((3, v), -torch.inf, dtype=dtype, device="cuda")
    one[:, v - 1] = 1.5
    r = call(one, np.array([0.0, 0.5, 0.999999], np.float32), draw_params(3, rng))
    assert (r.ids == v - 1).all() and (r.kept == 1).all() and (r.logprobs == 0).all()


def test_uniforms_at_the_ends(cuda_device):
    rng = np.random.default_rng(8)
    logits = rows(40, 3000, F32, rng)
    for u in (0.0, np.float32(1) - np.float32(2) ** -24, np.float32(1e-38)):
        p, us = draw_params(40, rng), np.full(40, u, np.float32)
        check(call(logits, us, p), logits, us, p)


def test_many_candidates(cuda_device):
    # as many as a row's room holds, one more, and far more: the same draw on either path
    rng = np.random.default_rng(9)
    for n in (2047, 2048, 2049, 5000):
        x = torch.full((2, 30000), -20.0, device="cuda")
        x[:, torch.from_numpy(rng.permutation(30000)[:n]).cuda()] = torch.from_numpy(rng.random((2, n)).astype(np.float32)).cuda()
        p = draw_params(2, rng, "plain")
        p["min_p"][:], p["temperature"][:] = 0.2, 1.0
        u = rng.random(2, dtype=np.float32)
        r = call(x, u, p)
        check(r, x, u, p)
        assert (r.kept == n).all()


def test_a_rising_row(cuda_device):
    # every logit is a new maximum: all of them pass the bound of their moment
    x = torch.linspace(-30, 30, 60000, device="cuda").expand(3, 60000)
    rng = np.random.default_rng(10)
    for src in (x, x.flip(1)):
        p, u = draw_params(3, rng, "plain"), rng.random(3, dtype=np.float32)
        check(call(src, u, p), src, u, p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("pad,shift", [(0, 1), (5, 0), (8, 3)])
def test_strides(cuda_device, dtype, pad, shift):
    rng = np.random.default_rng(11)
    n, v = 9, 3001
    room = torch.full((n * (v + pad) + 16,), 60.0, dtype=dtype, device="cuda")    # larger than any logit
    logits = room[shift:shift + n * (v + pad)].view(n, v + pad)[:, :v]
    logits.copy_(rows(n, v, dtype, rng))
    u, p = rng.random(n, dtype=np.float32), draw_params(n, rng)
    check(call(logits, u, p), logits, u, p)
    t = logits.t().contiguous().t()                        # columns first
    a, b = call(logits, u, p), call(t, u, p)
    assert torch.equal(a.ids, b.ids)
    assert torch.equal(call(logits[3:4].expand(4, v), u[:4], {k: q[:4] for k, q in p.items()}).ids[:1],
                       call(logits[3:4], u[:1], {k: q[:1] for k, q in p.items()}).ids)


def test_errors(cuda_device):
    x = torch.zeros(10, 500, device="cuda")
    x[0, 3], x[1, 4], x[2] = torch.nan, torch.inf, -torch.inf
    u = np.full(10, 0.5, np.float32)
    p = {"min_p": np.full(10, 0.1, np.float32), "temperature": np.ones(10, np.float32), "top_k": np.zeros(10, int),
         "top_p": np.ones(10, np.float32), "greedy": np.zeros(10, bool)}
    p["min_p"][3], p["min_p"][4], p["temperature"][5], p["top_p"][6] = 1.5, np.nan, -1.0, 0.0
    u[7] = 1.0
    want = [_lib.FG_ROW_NAN, _lib.FG_ROW_POS_INF, _lib.FG_ROW_ALL_MASKED] + [_lib.FG_ROW_BAD_PARAM] * 4 + \
        [_lib.FG_ROW_BAD_UNIFORM, 0, 0]
    for q in (0.1, 0.0):                                   # candidates, and the whole row
        p["min_p"][[0, 1, 2, 5, 6, 7, 8]] = q
        r = call(x, u, p)
        assert (r.status.cpu().numpy() & _lib.FG_ROW_ERROR_MASK).tolist() == want
        assert (r.ids[:8] == -1).all() and r.logprobs[:8].isnan().all() and (r.kept[:8] == 0).all()
        assert (r.ids[8:] >= 0).all()
        with pytest.raises(RuntimeError, match="nan"):
            call(x, u, p, check_errors=True)
    # greedy rows take what there is
    p["greedy"][:3] = True
    r = call(x, u, p)
    assert r.ids[:3].tolist() == [3, 4, 0] and (r.status[:3].cpu().numpy() & _lib.FG_ROW_ERROR_MASK == 0).all()
    # history ids outside the vocabulary are skipped and marked
    h = [[1, 2, 500]] + [[3, -1]] + [[] for _ in range(8)]
    r = call(x, u, p, {"rep": np.full(10, 1.1, np.float32)}, h)
    assert (r.status[:2].cpu().numpy() & _lib.FG_ROW_BAD_HISTORY != 0).all() and r.ids[1] == 4
    for kw in ({"min_p": torch.zeros(9, device="cuda")}, {"min_p": torch.zeros(10)}):
        with pytest.raises(ValueError, match="min_p"):
            sample_min_p(x, torch.zeros(10, device="cuda"), **kw)
    with pytest.raises(TypeError, match="top_k"):
        sample_min_p(x, torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda"), top_k=torch.zeros(10, device="cuda"))
    with pytest.raises(ValueError, match="longest"):
        sample_min_p(x, torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda"),
                     history=(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(11, dtype=torch.int64, device="cuda"), -1))


def test_without_min_p_it_is_fg_sample(cuda_device):
    # the batch of configuration 3 at 200 rows: the same chain, another kernel
    w = make_workload(3, batch=200, seed=3)
    p = w.params
    params = [SamplingParams(temperature=float(p.temperature[i]), top_p=float(p.top_p[i]), top_k=int(p.top_k[i]),
                             repetition_penalty=float(p.repetition_penalty[i]),
                             presence_penalty=float(p.presence_penalty[i]),
                             frequency_penalty=float(p.frequency_penalty[i]), greedy=bool(p.greedy[i]))
              for i in range(200)]
    logits, u = w.logits.cuda(), torch.from_numpy(w.uniforms).cuda()
    s = Sampler()
    want = s.sample(logits, params, token_histories=w.histories(), uniforms=u)
    # (one row of 201 with min-p takes the batch to the other entry point)
    more = torch.cat([logits, logits[:1]])
    got = s.sample(more, params + [SamplingParams(min_p=0.1)], token_histories=w.histories() + [[]],
                   uniforms=torch.cat([u, u[:1]]))
    # fg_sample's masses are 32-bit exponentials: a draw within 1e-6 of a border may differ
    assert (got[:200] != want).sum() <= 1


def test_kept_probabilities(cuda_device):
    rng = np.random.default_rng(12)
    for dtype, v in ((F32, 2000), (BF16, 70001)):
        logits, u, p = rows(30, v, dtype, rng), rng.random(30, dtype=np.float32), draw_params(30, rng)
        params = [SamplingParams(min_p=float(p["min_p"][i]), temperature=float(p["temperature"][i]),
                                 top_k=int(p["top_k"][i]), top_p=float(p["top_p"][i]), greedy=bool(p["greedy"][i]))
                  for i in range(30)]
        s = Sampler()
        ids = s.sample(logits, params, uniforms=torch.from_numpy(u).cuda(), return_probs=True)
        probs = s.last_probs.double().cpu().numpy()
        x = logits.float().cpu().numpy()
        for i in range(30):
            want = sample_row(x[i], u[i], p["min_p"][i], p["temperature"][i], p["top_k"][i], p["top_p"][i], p["greedy"][i])
            if want.near:
                continue
            assert int(ids[i]) == want.id
            full = np.zeros(v)
            full[want.kept_ids] = want.probs
            assert (np.abs(probs[i] - full) <= 1e-6 * full + 1e-12).all()
            assert ((probs[i] > 0) <= (full > 0)).all()


def test_the_decode_loop_and_host_buffers(cuda_device):
    rng = np.random.default_rng(13)
    n, v = 12, 4000
    params = [SamplingParams(min_p=[0.0, 0.05, 0.2][i % 3], temperature=0.9, top_k=[0, 40][i % 2],
                             repetition_penalty=1.2, frequency_penalty=0.3) for i in range(n)]
    dec = DecodeBatch(params, vocab=v, capacity=64, device="cuda", check_errors=True)
    history = [rng.integers(0, v, 5).tolist() for _ in range(n)]
    for i, h in enumerate(history):
        dec.set_history(i, h)
    for _ in range(6):
        logits, u = rows(n, v, BF16, rng, 1.5), rng.random(n, dtype=np.float32)
        ids = dec.step(logits, uniforms=torch.from_numpy(u).cuda()).tolist()
        x = logits.float().cpu().numpy()
        for i in range(n):
            q = params[i]
            want = sample_row(x[i], u[i], q.min_p, q.temperature, q.top_k, q.top_p, rep=q.repetition_penalty,
                              freq=q.frequency_penalty, history=history[i])
            assert want.near or ids[i] == want.id
            history[i].append(ids[i])
    assert dec.histories() == history
    # a later batch without min-p on the same stream: fg_sample's counters are untouched
    w = make_workload(2, batch=8, seed=1)
    want = Sampler().sample(w.logits.cuda(), [SamplingParams()] * 8, uniforms=torch.from_numpy(w.uniforms).cuda())
    assert torch.equal(want, Sampler().sample(w.logits.cuda(), [SamplingParams()] * 8, uniforms=torch.from_numpy(w.uniforms).cuda()))
    # host buffers
    w = make_workload(2, batch=16, seed=2)
    w.params.min_p = np.full(16, 0.1, np.float32)
    host = HostBatchSampler(16, w.vocab, w.logits.dtype, w.hist_ids.size, "cuda")
    ids = host.sample(w.logits.pin_memory(), w.params, torch.from_numpy(w.hist_ids).pin_memory(),
                      torch.from_numpy(w.hist_offsets).pin_memory(), w.uniforms, w.hist_max_len)
    torch.cuda.synchronize()
    x, hs = w.logits.float().numpy(), w.histories()
    for i in range(16):
        want = sample_row(x[i], w.uniforms[i], 0.1, 0.7, 50, 0.95, rep=1.1, pres=0.2, freq=0.1, history=hs[i])
        assert want.near or int(ids[i]) == want.id


def test_streams_and_graphs(cuda_device):
    rng = np.random.default_rng(14)
    logits, u, p = rows(30, 9000, BF16, rng), rng.random(30, dtype=np.float32), draw_params(30, rng)
    history = [rng.integers(0, 9000, 100) for _ in range(30)]
    pen = {"rep": np.full(30, 1.2, np.float32)}
    want = call(logits, u, p, pen, history)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = call(logits, u, p, pen, history)
    torch.cuda.synchronize()
    assert torch.equal(got.ids, want.ids) and torch.equal(got.logprobs, want.logprobs)
    us, ms = torch.from_numpy(u).cuda(), torch.from_numpy(p["min_p"]).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = sample_min_p(logits, us, ms)
    for seed in (1, 2):
        u2 = np.random.default_rng(seed).random(30, dtype=np.float32)
        logits.copy_(rows(30, 9000, BF16, np.random.default_rng(seed)))
        us.copy_(torch.from_numpy(u2))
        graph.replay()
        torch.cuda.synchronize()
        q = {"min_p": p["min_p"], "temperature": np.ones(30, np.float32), "top_k": np.zeros(30, int),
             "top_p": np.ones(30, np.float32), "greedy": np.zeros(30, bool)}
        check(r, logits, u2, q)


def test_two_threads(cuda_device):
    # sizes that need different amounts of shared memory, with histories and without, side by side
    import threading

    rng = np.random.default_rng(15)
    jobs = []
    for v, h in ((700, 0), (5000, 40), (20000, 1500), (40000, 0), (70000, 4000), (9000, 9)):
        logits, u, p = rows(6, v, F32, rng), rng.random(6, dtype=np.float32), draw_params(6, rng)
        history = [rng.integers(0, v, h) for _ in range(6)] if h else None
        pen = {"rep": np.full(6, 1.3, np.float32)} if h else None
        jobs.append((logits, u, p, pen, history))
    torch.cuda.synchronize()
    got, start = [None] * len(jobs), threading.Barrier(len(jobs))

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait(timeout=60)
            got[i] = [call(*jobs[i]) for _ in range(5)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for job, results in zip(jobs, got):
        assert results is not None
        for r in results:
            check(r, *job)


def test_no_rows(cuda_device):
    r = sample_min_p(torch.zeros(0, 50, device="cuda"), torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda"))
    assert r.ids.shape == (0,) and r.logprobs.shape == (0,)


def test_frequencies(cuda_device):
    # 40000 uniforms of one row: each token's share is its probability (5 standard deviations)
    x = torch.tensor([2.0, 1.0, 0.5, 0.0, -1.0, -9.0], device="cuda").expand(40000, 6)
    u = (torch.arange(40000, device="cuda", dtype=F32) + 0.5) / 40000
    ids = sample_min_p(x, u, torch.full((40000,), 0.1, device="cuda")).ids
    p = torch.softmax(torch.tensor([2.0, 1.0, 0.5, 0.0]), 0)
    share = torch.bincount(ids, minlength=6).cpu() / 40000
    assert (share[4:] == 0).all() and (share[:4] - p).abs().max() <= 2 / 40000
