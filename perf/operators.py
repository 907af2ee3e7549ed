"""The operators around the sampler: what is measured, in plain form and through the package.

* ``logprobs``: log probabilities of given tokens with the rows' entropy, the tokens' ranks and the
  top alternatives (``token_logprobs``).
* ``gradient``: the gradient of those log probabilities and entropies with respect to the logits
  (``token_logprobs_grad``).
* ``adapters``: an LM head shared by a batch of requests, with each request's own low-rank adapter
  beside it (``AdapterHead.logits``).

With ``own`` false ``run`` evaluates the definitions with elementary torch operations in 32 bits;
with ``own`` true it makes the calls a user of the package makes.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one sequence being decoded, the largest vocabulary: latency of a served logprob request
        {"name": "logprobs-1x256000-f32-top20", "op": "logprobs", "rows": 1, "vocab": 256000, "dtype": "f32",
         "top": 20, "tempered": True, "masked": False, "pad": 0},
        # an ordinary serving batch with structured output: a third of the rows under a grammar mask
        {"name": "logprobs-256x32000-f16-top5-masked", "op": "logprobs", "rows": 256, "vocab": 32000, "dtype": "f16",
         "top": 5, "tempered": True, "masked": True, "pad": 0},
        # a large serving batch, every request asking for the alternatives
        {"name": "logprobs-1024x128256-bf16-top20", "op": "logprobs", "rows": 1024, "vocab": 128256, "dtype": "bf16",
         "top": 20, "tempered": True, "masked": False, "pad": 0},
        # a prompt being scored: odd row count, odd vocabulary (no row but the first is 16-byte aligned)
        {"name": "logprobs-777x50257-bf16-top1", "op": "logprobs", "rows": 777, "vocab": 50257, "dtype": "bf16",
         "top": 1, "tempered": False, "masked": False, "pad": 0},
        # a trainer rescoring rollouts: only the tokens' own log probabilities and the entropies
        {"name": "logprobs-4096x152064-f32", "op": "logprobs", "rows": 4096, "vocab": 152064, "dtype": "f32",
         "top": 0, "tempered": True, "masked": False, "pad": 0},
        # the smallest training step: one short completion
        {"name": "gradient-8x50257-f32", "op": "gradient", "rows": 8, "vocab": 50257, "dtype": "f32",
         "tempered": False, "masked": False, "entropy": False, "pad": 0},
        # an ordinary loss-scaled step on a padded (strided) logits buffer with an odd vocabulary
        {"name": "gradient-333x32001-f16-entropy", "op": "gradient", "rows": 333, "vocab": 32001, "dtype": "f16",
         "tempered": True, "masked": True, "entropy": True, "pad": 63},
        # a policy-gradient step with an entropy bonus over a packed batch
        {"name": "gradient-1024x128256-bf16-entropy", "op": "gradient", "rows": 1024, "vocab": 128256,
         "dtype": "bf16", "tempered": True, "masked": False, "entropy": True, "pad": 0},
        # one request decoding with its adapter: the weight is read for a single token
        {"name": "adapters-1x4096x128256-bf16-r16", "op": "adapters", "rows": 1, "dim": 4096, "vocab": 128256,
         "dtype": "bf16", "out": "f32", "rank": 16, "slots": 8, "bare": False},
        # many tenants in one ordinary batch
        {"name": "adapters-64x2048x32000-f16-r8", "op": "adapters", "rows": 64, "dim": 2048, "vocab": 32000,
         "dtype": "f16", "out": "f16", "rank": 8, "slots": 32, "bare": True},
        # odd everywhere: rows, width, vocabulary and rank
        {"name": "adapters-37x1001x50257-bf16-r20", "op": "adapters", "rows": 37, "dim": 1001, "vocab": 50257,
         "dtype": "bf16", "out": "bf16", "rank": 20, "slots": 5, "bare": True},
        # the largest decode batch
        {"name": "adapters-1024x4096x128256-bf16-r16", "op": "adapters", "rows": 1024, "dim": 4096, "vocab": 128256,
         "dtype": "bf16", "out": "bf16", "rank": 16, "slots": 16, "bare": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "gradient", "adapters"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "adapters":
        dtype = rng.choice(["f16", "bf16"])
        dim = rng.choice([512, 1024, 2048, 4096]) - rng.choice([0, rng.randint(1, 255)])
        if rng.random() < 0.7:
            dim = dim // 8 * 8
        return {"op": op, "rows": _log_int(rng, 1, 1024), "dim": dim, "vocab": rng.randint(32000, 128256),
                "dtype": dtype, "out": rng.choice([dtype, "f32"]), "rank": rng.randint(4, 64),
                "slots": rng.randint(1, 16), "bare": rng.random() < 0.5}
    vocab = _log_int(rng, 32000, 256000)
    limit = 4096 * 152064 * 4 // (vocab * _BYTES[dtype])
    if op == "gradient":
        limit = 1024 * 128256 * 2 // (vocab * _BYTES[dtype])
    case = {"op": op, "rows": min(_log_int(rng, 1, 3000), limit), "vocab": vocab, "dtype": dtype,
            "tempered": rng.random() < 0.5, "masked": rng.random() < 0.3, "pad": rng.choice([0, 0, 1, 56])}
    if op == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20, 32])
    else:
        case["entropy"] = rng.random() < 0.5
    return case


# ---- inputs -------------------------------------------------------------------------------------

def _logits_state(case, gen):
    n, v = case["rows"], case["vocab"]
    dtype = _DTYPES[case["dtype"]]
    dev = "cuda"
    buf = torch.empty(n, v + case["pad"], dtype=dtype, device=dev)
    step = max(1, (1 << 27) // (v + case["pad"]))
    for lo in range(0, n, step):   # N(0,1) with a peaked head: +8 on 1 % of the ids
        part = torch.randn(min(step, n - lo), v + case["pad"], device=dev, generator=gen)
        part += 8.0 * (torch.rand(part.shape, device=dev, generator=gen) < 0.01)
        buf[lo:lo + part.shape[0]] = part.to(dtype)
    logits = buf[:, :v]
    # given tokens: likely ones (the best of 64 random ids), and some rows without a token
    ids = torch.randint(0, v, (n, 64), device=dev, generator=gen)
    best = logits.gather(1, ids).float().argmax(dim=1, keepdim=True)
    tokens = ids.gather(1, best)[:, 0]
    if case["masked"]:
        # every third row keeps 100 ids; the others are -inf, or the type's lowest value in every sixth row
        for r in range(0, n, 3):
            keep = torch.randint(0, v, (100,), device=dev, generator=gen)
            row = torch.full((v,), -math.inf if r % 2 else torch.finfo(dtype).min, dtype=dtype, device=dev)
            row[keep] = logits[r, keep]
            logits[r] = row
            tokens[r] = keep[0]
    tokens = torch.where(torch.rand(n, device=dev, generator=gen) < 0.05, torch.full_like(tokens, -1), tokens)
    temperature = None
    if case["tempered"]:
        temperature = 0.5 + 0.7 * torch.rand(n, device=dev, generator=gen)
    return {"logits": logits, "tokens": tokens, "temperature": temperature}


def _row_max_logsum(logits, temperature):
    n, v = logits.shape
    top = torch.empty(n, dtype=torch.float32, device=logits.device)
    logsum = torch.empty_like(top)
    step = max(1, (1 << 27) // v)
    for lo in range(0, n, step):
        x = logits[lo:lo + step].double()
        m = x.max(dim=1).values
        y = x - m[:, None]
        if temperature is not None:
            y = y / temperature[lo:lo + step, None].double()
        top[lo:lo + step] = m.float()
        logsum[lo:lo + step] = y.exp().sum(dim=1).log().float()
    return top, logsum


def _entropies(logits, temperature, top, logsum):
    n, v = logits.shape
    out = torch.empty(n, dtype=torch.float32, device=logits.device)
    step = max(1, (1 << 27) // v)
    for lo in range(0, n, step):
        y = logits[lo:lo + step].double() - top[lo:lo + step, None].double()
        if temperature is not None:
            y = y / temperature[lo:lo + step, None].double()
        lp = y - logsum[lo:lo + step, None].double()
        p = lp.exp()
        out[lo:lo + step] = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(dim=1).float()
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] in ("logprobs", "gradient"):
        state.update(_logits_state(case, gen))
        if case["op"] == "gradient":
            # what the forward pass left: each row's maximum, log sum and entropy; and the loss's gradients,
            # scaled in 16-bit floats as a loss scaler does
            n = case["rows"]
            state["top"], state["logsum"] = _row_max_logsum(state["logits"], state["temperature"])
            state["entropy"] = _entropies(state["logits"], state["temperature"], state["top"], state["logsum"])
            scale = 1024.0 if case["dtype"] == "f16" else 1.0
            state["grad_logprobs"] = torch.randn(n, device="cuda", generator=gen) * scale
            state["grad_entropy"] = None
            if case["entropy"]:
                state["grad_entropy"] = torch.full((n,), 0.01 * scale, device="cuda")
        return state
    dtype = _DTYPES[case["dtype"]]
    b, d, v, r, s = case["rows"], case["dim"], case["vocab"], case["rank"], case["slots"]

    def normal(shape, scale):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)

    weight = normal((v, d), d ** -0.5)
    state["hidden"] = normal((b, d), 1.0)
    a = [normal((r, d), d ** -0.5) for _ in range(s)]
    up = [normal((v, r), 0.1) for _ in range(s)]
    scales = [0.5 + 0.25 * (i % 4) for i in range(s)]
    low = -1 if case["bare"] else 0   # -1: a request without an adapter
    state["adapters"] = torch.randint(low, s, (b,), device="cuda", generator=gen, dtype=torch.int32)
    state["out"] = _DTYPES[case["out"]]
    if own:
        from flashgen_b200.sampling.lm_head import AdapterHead
        head = AdapterHead(weight, slots=s, rank=r)
        for i in range(s):
            head.load(i, a[i], up[i], scales[i])
        state["head"] = head
    else:
        state.update(weight=weight, down=torch.stack(a), up=torch.stack(up),
                     scales=torch.tensor(scales, device="cuda"))
    return state


# ---- one pass -----------------------------------------------------------------------------------

def _tempered(x, temperature):
    return x if temperature is None else x / temperature[:, None]


def _plain_logprobs(s):
    x = s["logits"].float()
    n, v = x.shape
    tokens, k = s["tokens"], s["case"]["top"]
    top = x.max(dim=1).values
    y = _tempered(x - top[:, None], s["temperature"])
    e = y.exp()
    total = e.sum(dim=1)
    logsum = total.log()
    entropy = logsum - torch.where(e > 0, e * y, torch.zeros_like(e)).sum(dim=1) / total
    del e
    given = tokens >= 0
    at = tokens.clamp_min(0)[:, None]
    lp = torch.where(given, y.gather(1, at)[:, 0] - logsum, torch.zeros_like(logsum))
    xt = x.gather(1, at)
    ids = torch.arange(v, device=x.device)[None, :]
    rank = ((x > xt) | ((x == xt) & (ids < at))).sum(dim=1).to(torch.int32)
    out = {"logprobs": lp, "entropy": entropy, "top": top, "logsum": logsum,
           "rank": torch.where(given, rank, torch.full_like(rank, -1))}
    if k > 0:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        out["top_ids"] = order
        out["top_logprobs"] = y.gather(1, order) - logsum[:, None]
    return out


def _plain_gradient(s):
    x = s["logits"].float()
    y = _tempered(x - s["top"][:, None], s["temperature"]) - s["logsum"][:, None]
    del x
    p = y.exp()
    g = torch.where(s["tokens"] >= 0, s["grad_logprobs"], torch.zeros_like(s["grad_logprobs"]))
    d = -g[:, None] * p
    if s["grad_entropy"] is not None:
        h = s["grad_entropy"][:, None]
        d = d - torch.where(p > 0, h * p * (y + s["entropy"][:, None]), torch.zeros_like(p))
    d.scatter_add_(1, s["tokens"].clamp_min(0)[:, None], g[:, None])
    return {"grad_logits": _tempered(d, s["temperature"]).to(s["logits"].dtype)}


def _plain_adapters(s):
    x = s["hidden"].float()
    out = x @ s["weight"].float().T
    for i in range(s["down"].shape[0]):
        mine = (s["adapters"] == i).to(torch.float32)[:, None]
        u = (x @ s["down"][i].float().T) * s["scales"][i] * mine
        out += u @ s["up"][i].float().T
    return {"logits": out.to(s["out"])}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"logprobs": _plain_logprobs, "gradient": _plain_gradient, "adapters": _plain_adapters}[op](state)
    if op == "adapters":
        return {"logits": state["head"].logits(state["hidden"], state["adapters"], out_dtype=state["out"])}
    from flashgen_b200.sampling.logprobs import token_logprobs, token_logprobs_grad
    if op == "gradient":
        grad = token_logprobs_grad(state["logits"], state["tokens"], state["top"], state["logsum"],
                                   state["grad_logprobs"], entropy=state["entropy"],
                                   grad_entropy=state["grad_entropy"], temperature=state["temperature"])
        return {"grad_logits": grad}
    r = token_logprobs(state["logits"], state["tokens"], temperature=state["temperature"], top=state["case"]["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy, "top": r.max, "logsum": r.logsum, "rank": r.rank}
    if state["case"]["top"] > 0:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


def work(case):
    if case["op"] == "adapters":
        b, d, v, r = case["rows"], case["dim"], case["vocab"], case["rank"]
        esz = _BYTES[case["dtype"]]
        used = min(case["slots"], b)
        return {"bytes": esz * (b * d + v * d + used * r * (d + v)) + 4 * b + b * v * _BYTES[case["out"]],
                "flops": 2 * b * v * d + 2 * b * r * (d + v)}
    n, v = case["rows"], case["vocab"]
    esz = _BYTES[case["dtype"]]
    if case["op"] == "gradient":
        return {"bytes": 2 * n * v * esz + n * 28, "flops": 6 * n * v}
    return {"bytes": n * v * esz + n * (8 + 4 + 20 + 12 * case["top"]), "flops": 6 * n * v}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def _exact_rows(state, lo, hi):
    """Log probabilities [hi - lo, V] of rows lo..hi in 64 bits, and their maxima and log sums."""
    x = state["logits"][lo:hi].to(torch.float64)
    t = state["temperature"]
    inv = torch.ones(hi - lo, 1, dtype=torch.float64, device=x.device)
    if t is not None:
        inv = 1.0 / t[lo:hi, None].to(torch.float64)
    peak = torch.amax(x, dim=1, keepdim=True)
    logsum = torch.log(torch.sum(torch.exp((x - peak) * inv), dim=1, keepdim=True))
    return x, (x - peak) * inv - logsum, peak[:, 0], logsum[:, 0], inv


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = keep
    if case["op"] == "adapters":
        x = state["hidden"].double()
        b, v = case["rows"], case["vocab"]
        out = torch.empty(b, v, dtype=torch.float64, device="cuda")
        slot = state["adapters"].long()
        u = torch.zeros(b, case["rank"], dtype=torch.float64, device="cuda")
        for r in range(b):
            if int(slot[r]) >= 0:
                u[r] = state["down"][slot[r]].double().mv(x[r]) * float(state["scales"][slot[r]])
        for lo in range(0, v, 16384):
            part = x @ state["weight"][lo:lo + 16384].double().T
            for i in range(case["slots"]):
                rows = torch.nonzero(slot == i)[:, 0]
                if rows.numel():
                    part[rows] += u[rows] @ state["up"][i, lo:lo + 16384].double().T
            out[:, lo:lo + 16384] = part
        return {"logits": out}
    n, v = case["rows"], case["vocab"]
    step = max(1, (1 << 26) // v)
    parts = []
    for lo in range(0, n, step):
        hi = min(n, lo + step)
        x, lp, peak, logsum, inv = _exact_rows(state, lo, hi)
        p = torch.exp(lp)
        plogp = torch.xlogy(p, p)
        h = -plogp.sum(dim=1)
        tokens = state["tokens"][lo:hi]
        rows = torch.arange(hi - lo, device="cuda")
        given = tokens >= 0
        at = tokens.clamp_min(0)
        if case["op"] == "gradient":
            g = torch.where(given, state["grad_logprobs"][lo:hi].double(), 0.0)
            d = -g[:, None] * p
            if state["grad_entropy"] is not None:
                d = d - state["grad_entropy"][lo:hi, None].double() * (plogp + p * h[:, None])
            d[rows, at] += g
            parts.append({"grad_logits": d * inv})
            continue
        xt = x[rows, at]
        ahead = (x > xt[:, None]).sum(dim=1)
        same = x == xt[:, None]
        same &= torch.arange(v, device="cuda")[None, :] < at[:, None]
        ahead += same.sum(dim=1)
        part = {"logprobs": torch.where(given, lp[rows, at], 0.0), "entropy": h, "top": peak, "logsum": logsum,
                "rank": torch.where(given, ahead, -1).to(torch.int32)}
        if case["top"] > 0:
            # the order of values, then of ids: a stable descending sort
            order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case["top"]]
            part["top_ids"] = order
            part["top_logprobs"] = lp.gather(1, order)
        parts.append(part)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
