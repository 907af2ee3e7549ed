"""More operators around the sampler: what is measured, in plain form and through the package.

* ``sample``: one token a row with penalties, temperature, min-p, top-k and top-p, from given uniforms; with the drawn
  id's log probability among the tokens that were kept, and their number (``sample_min_p``).
* ``linear``: ``act(x W^T + b) + residual``, the dense block in front of an LM head; as a serving call, and as a
  training step with the gradients of everything that goes in (``fused_linear``).
* ``clip``: the global norm of a list of gradients and the gradients scaled to at most a given norm
  (``clip_grad_norm``).

With ``own`` false ``run`` evaluates the definitions with elementary torch operations in 32 bits (probabilities and the
long sums in 64); with ``own`` true it makes the calls a user of the package makes.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_MOST_LOGITS = 1024 * 128256
_MOST_PRODUCT = 8192 * 4096 * 4096
_MOST_GRADS = 48 * 4096 * 4096


def listed():
    return [
        # one sequence being decoded with the largest vocabulary: the latency of a step
        {"name": "sample-1x256000-f32", "op": "sample", "rows": 1, "vocab": 256000, "dtype": "f32", "mixed": False,
         "history": 0, "masked": False, "pad": 0},
        # a small serving batch with penalties over its histories; odd rows and an odd vocabulary
        {"name": "sample-37x50257-f16-history", "op": "sample", "rows": 37, "vocab": 50257, "dtype": "f16",
         "mixed": True, "history": 700, "masked": False, "pad": 0},
        # an ordinary batch whose requests bring their own parameters, some under a grammar mask
        {"name": "sample-256x32000-bf16-masked", "op": "sample", "rows": 256, "vocab": 32000, "dtype": "bf16",
         "mixed": True, "history": 0, "masked": True, "pad": 24},
        # a large serving batch with one sampling preset
        {"name": "sample-1024x128256-bf16", "op": "sample", "rows": 1024, "vocab": 128256, "dtype": "bf16",
         "mixed": False, "history": 0, "masked": False, "pad": 0},
        # a large batch of requests with their own parameters, histories included
        {"name": "sample-512x128256-bf16-mixed", "op": "sample", "rows": 512, "vocab": 128256, "dtype": "bf16",
         "mixed": True, "history": 1024, "masked": False, "pad": 0},
        # the block in front of the head for one sequence being decoded
        {"name": "linear-1x4096x4096-bf16", "op": "linear", "tokens": 1, "inner": 4096, "outer": 4096,
         "dtype": "bf16", "act": "silu", "bias": True, "residual": True, "train": False},
        # a prompt's hidden states through the block
        {"name": "linear-1024x4096x4096-bf16", "op": "linear", "tokens": 1024, "inner": 4096, "outer": 4096,
         "dtype": "bf16", "act": "silu", "bias": True, "residual": True, "train": False},
        # a training step over a ragged batch; no size a multiple of anything
        {"name": "linear-777x1001x2050-f16-train", "op": "linear", "tokens": 777, "inner": 1001, "outer": 2050,
         "dtype": "f16", "act": "gelu", "bias": True, "residual": False, "train": True},
        # a training step over a full batch
        {"name": "linear-8192x4096x4096-bf16-train", "op": "linear", "tokens": 8192, "inner": 4096, "outer": 4096,
         "dtype": "bf16", "act": "silu", "bias": True, "residual": True, "train": True},
        # one tenant's adapter: two small matrices
        {"name": "clip-2-bf16", "op": "clip", "tensors": 2, "rows": 32000, "cols": 16, "dtype": "bf16",
         "out": "f32", "small": 65536},
        # a bank of adapters with a bias or a scale beside each
        {"name": "clip-60-f32", "op": "clip", "tensors": 60, "rows": 32000, "cols": 16, "dtype": "f32", "out": "f32",
         "small": 16},
        # the blocks of a large network, into the optimizer's 32-bit gradients
        {"name": "clip-48-bf16", "op": "clip", "tensors": 48, "rows": 4096, "cols": 4096, "dtype": "bf16",
         "out": "f32", "small": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "linear", "clip"])
    if op == "sample":
        vocab = _log_int(rng, 32000, 256000)
        return {"op": op, "rows": min(_log_int(rng, 1, 1024), _MOST_LOGITS // 2 // vocab), "vocab": vocab,
                "dtype": rng.choice(["f32", "f16", "bf16"]), "mixed": rng.random() < 0.5,
                "history": rng.choice([0, 0, _log_int(rng, 1, 2000)]), "masked": rng.random() < 0.3,
                "pad": rng.choice([0, 0, 1, 56])}
    if op == "linear":
        inner, outer = _log_int(rng, 256, 4096), _log_int(rng, 256, 4096)
        if rng.random() < 0.6:
            inner, outer = (inner + 63) // 64 * 64, (outer + 63) // 64 * 64
        return {"op": op, "tokens": min(_log_int(rng, 1, 8192), _MOST_PRODUCT // (inner * outer)), "inner": inner,
                "outer": outer, "dtype": rng.choice(["f16", "bf16"]),
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.5, "train": rng.random() < 0.5}
    tensors = _log_int(rng, 1, 60)
    rows, cols = _log_int(rng, 16, 32000), _log_int(rng, 8, 4096)
    rows = max(1, min(rows, _MOST_GRADS // (tensors * cols)))
    dtype = rng.choice(["f32", "f16", "bf16"])
    return {"op": op, "tensors": tensors, "rows": rows, "cols": cols, "dtype": dtype, "out": rng.choice([dtype, "f32"]),
            "small": rng.choice([0, 1, 16, 4097])}


# ---- inputs -------------------------------------------------------------------------------------

def _sample_state(case, gen):
    n, v = case["rows"], case["vocab"]
    dtype = _DTYPES[case["dtype"]]
    dev = "cuda"

    def uniform(*shape):
        return torch.rand(shape, device=dev, generator=gen)

    buf = torch.empty(n, v + case["pad"], dtype=dtype, device=dev)
    step = max(1, (1 << 27) // (v + case["pad"]))
    for lo in range(0, n, step):   # rows from sure to unsure: normal logits of standard deviation 1.5 to 3.5
        part = torch.randn(min(step, n - lo), v + case["pad"], device=dev, generator=gen)
        part *= 1.5 + 2.0 * uniform(part.shape[0], 1)
        buf[lo:lo + part.shape[0]] = part.to(dtype)
    logits = buf[:, :v]
    if case["masked"]:
        # every third row keeps some 100 ids; the others are -inf, or the type's lowest value in every sixth row
        keep = uniform((n + 2) // 3, v) < 100.0 / v
        keep[:, 5] = True
        low = torch.full(((n + 2) // 3, 1), -math.inf, device=dev)
        low[1::2] = torch.finfo(dtype).min
        logits[::3] = torch.where(keep, logits[::3], low.to(dtype))
    s = {"logits": logits, "uniforms": uniform(n), "temperature": 0.6 + 0.7 * uniform(n),
         "min_p": torch.full((n,), 0.05, device=dev), "top_k": None, "top_p": None, "greedy": None,
         "repetition": None, "presence": None, "frequency": None, "history": None}
    if case["mixed"]:
        s["min_p"] = torch.tensor([0.02, 0.05, 0.1, 0.3], device=dev)[torch.randint(0, 4, (n,), device=dev, generator=gen)]
        s["top_k"] = torch.tensor([0, 20, 100, 1000], device=dev)[torch.randint(0, 4, (n,), device=dev, generator=gen)].to(torch.int32)
        s["top_p"] = torch.where(uniform(n) < 0.5, 0.8 + 0.2 * uniform(n), torch.ones(n, device=dev))
        kind = uniform(n)
        s["greedy"] = kind > 0.95
        # a tenth of the requests without min-p: half of those with top-k, half with top-p alone
        none = kind < 0.1
        s["min_p"] = torch.where(none, torch.zeros_like(s["min_p"]), s["min_p"])
        s["top_k"] = torch.where(none, torch.where(kind < 0.05, torch.full_like(s["top_k"], 50), torch.zeros_like(s["top_k"])), s["top_k"])
        s["top_p"] = torch.where(none, torch.full_like(s["top_p"], 0.9), s["top_p"])
    if case["history"]:
        # what a decode loop keeps: the rows' ids one after the other, where each row begins, the longest
        longest = case["history"]
        lens = torch.randint(0, longest + 1, (n,), device=dev, generator=gen)
        offsets = torch.zeros(n + 1, dtype=torch.int64, device=dev)
        offsets[1:] = torch.cumsum(lens, 0)
        ids = (uniform(n * longest) ** 3 * v).to(torch.int32).clamp_(max=v - 1)   # low ids come back often
        s["history"] = (ids, offsets, longest)
        s["repetition"] = 1.0 + 0.2 * uniform(n)
        s["presence"] = 0.4 * uniform(n)
        s["frequency"] = 0.2 * uniform(n)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(shape, scale, kind=dtype):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(kind)

    if case["op"] == "sample":
        return {"case": case, **_sample_state(case, gen)}
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        s = {"case": case, "x": normal((m, k), 1.0), "weight": normal((n, k), k ** -0.5),
             "bias": normal((n,), 0.5) if case["bias"] else None,
             "residual": normal((m, n), 1.0) if case["residual"] else None}
        if case["train"]:
            s["grad"] = normal((m, n), 1.0)
            s["leaves"] = [s[name].requires_grad_() for name in ("x", "weight", "bias", "residual") if s[name] is not None]
        return s
    grads = []
    for i in range(case["tensors"]):
        # every second tensor of a list with a small one beside it is that small one
        shape = (case["rows"], case["cols"]) if not case["small"] or i % 2 == 0 else (case["small"],)
        grads.append(normal(shape, 1e-3 * (1 + i % 3)))
    return {"case": case, "grads": grads, "max_norm": 1.0,
            "out": [torch.empty_like(g, dtype=_DTYPES[case["out"]]) for g in grads]}


# ---- one pass -----------------------------------------------------------------------------------

def _plain_sample(s):
    x = s["logits"].float()
    n, v = x.shape
    if s["history"] is not None:
        ids, offsets, _ = s["history"]
        rows = torch.repeat_interleave(torch.arange(n, device=x.device), offsets[1:] - offsets[:-1])
        counts = torch.zeros(n, v, device=x.device)
        counts.index_put_((rows, ids[:rows.numel()].long()), torch.ones(1, device=x.device), accumulate=True)
        r, f, p = s["repetition"][:, None], s["frequency"][:, None], s["presence"][:, None]
        x = torch.where(counts > 0, torch.where(x > 0, x / r, x * r) - f * counts - p, x)
    y = x / s["temperature"][:, None] + 0.0
    ys, order = torch.sort(y, dim=1, descending=True, stable=True)
    d = ys.double() - ys[:, :1].double()
    keep = (d >= s["min_p"].double().log()[:, None]) & (ys > -math.inf)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"].clamp(max=v), torch.full_like(s["top_k"], v)).long()
        keep &= ys >= ys.gather(1, k[:, None] - 1)
    if s["greedy"] is not None:
        keep &= ~s["greedy"][:, None] | (torch.arange(v, device=x.device) == 0)
    mass = torch.where(keep, d.exp(), torch.zeros_like(d))
    upto = mass.cumsum(dim=1)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        keep &= (upto - mass <= p * mass.sum(dim=1, keepdim=True)) | (p >= 1)
        mass = torch.where(keep, mass, torch.zeros_like(mass))
    kept = keep.sum(dim=1)
    total = mass.sum(dim=1)
    at = (keep & (upto <= (s["uniforms"].double() * total)[:, None])).sum(dim=1).minimum(kept - 1)[:, None]
    return {"ids": order.gather(1, at)[:, 0], "logprobs": (mass.gather(1, at)[:, 0] / total).log().float(),
            "kept": kept.to(torch.int32)}


def _act(kind, z):
    """The activation of z and its derivative."""
    if kind == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    dtype = s["x"].dtype
    z = x @ w.T
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    out, slope = _act(case["act"], z)
    if s["residual"] is not None:
        out = out + s["residual"].detach().float()
    result = {"out": out.to(dtype)}
    if case["train"]:
        dz = s["grad"].float() * slope
        result["grad_x"], result["grad_weight"] = (dz @ w).to(dtype), (dz.T @ x).to(dtype)
        if s["bias"] is not None:
            result["grad_bias"] = dz.sum(dim=0).to(dtype)
        if s["residual"] is not None:
            result["grad_residual"] = s["grad"]
    return result


def _plain_clip(s):
    flat = [g.float() for g in s["grads"]]
    norm = torch.stack([torch.sum(g * g, dtype=torch.float64) for g in flat]).sum().sqrt().float()
    scale = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return {"norm": norm, "grads": [(g * scale).to(o.dtype) for g, o in zip(flat, s["out"])]}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"sample": _plain_sample, "linear": _plain_linear, "clip": _plain_clip}[op](state)
    if op == "sample":
        from flashgen_b200 import sample_min_p
        r = sample_min_p(state["logits"], state["uniforms"], state["min_p"], temperature=state["temperature"],
                         top_k=state["top_k"], top_p=state["top_p"], greedy=state["greedy"],
                         repetition_penalty=state["repetition"], presence_penalty=state["presence"],
                         frequency_penalty=state["frequency"], history=state["history"])
        return {"ids": r.ids, "logprobs": r.logprobs, "kept": r.kept}
    if op == "linear":
        from flashgen_b200 import fused_linear
        out = fused_linear(state["x"], state["weight"], state["bias"], state["residual"],
                           activation=state["case"]["act"])
        if not state["case"]["train"]:
            return {"out": out}
        grads = iter(torch.autograd.grad(out, state["leaves"], state["grad"]))
        names = [name for name in ("x", "weight", "bias", "residual") if state[name] is not None]
        return {"out": out.detach(), **{"grad_" + name: next(grads) for name in names}}
    from flashgen_b200 import clip_grad_norm
    norm = clip_grad_norm(state["grads"], state["max_norm"], out=state["out"])
    return {"norm": norm, "grads": state["out"]}


def work(case):
    esz = _BYTES[case["dtype"]]
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        # a comparison a logit; the kept tokens' exponentials are few beside it
        return {"bytes": n * v * esz + n * (4 * 3 + 9 * case["mixed"] + 8 + 4 + 4) +
                (n * (2 * case["history"] + 8 + 12) if case["history"] else 0), "flops": n * v}
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        read = m * k + n * k + n * case["bias"] + m * n * case["residual"]
        if case["train"]:   # the result's gradient in; the result and the gradients out
            return {"bytes": esz * (2 * read + 2 * m * n), "flops": 6 * m * n * k}
        return {"bytes": esz * (read + m * n), "flops": 2 * m * n * k}
    count = case["tensors"] * case["rows"] * case["cols"]
    if case["small"]:
        count = (case["tensors"] + 1) // 2 * case["rows"] * case["cols"] + case["tensors"] // 2 * case["small"]
    return {"bytes": count * (esz + _BYTES[case["out"]]), "flops": 3 * count}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def _exact_row(s, r):
    """The drawn id's log probability of one row, from the set of tokens that are kept."""
    x = s["logits"][r].to(torch.float32)
    if s["history"] is not None:
        ids, offsets, _ = s["history"]
        seen, times = torch.unique(ids[int(offsets[r]):int(offsets[r + 1])].long(), return_counts=True)
        old = x[seen]
        # the penalties are operations on 32-bit numbers, by the definition
        new = torch.where(old > 0, old / s["repetition"][r], old * s["repetition"][r])
        x = x.clone()
        x[seen] = new - s["frequency"][r] * times.to(torch.float32) - s["presence"][r]
    if s["greedy"] is not None and bool(s["greedy"][r]):
        return 0.0
    y = (x / s["temperature"][r]).double()
    least = y.max() + torch.log(s["min_p"][r].double())
    ids = torch.nonzero((y >= least) & (y > -math.inf))[:, 0]
    values = y[ids]
    if s["top_k"] is not None and 0 < int(s["top_k"][r]) < ids.numel():
        bound = torch.topk(values, int(s["top_k"][r])).values[-1]
        values = values[values >= bound]
    p = torch.softmax(values, 0).sort(descending=True).values
    if s["top_p"] is not None and float(s["top_p"][r]) < 1:
        before = torch.cat([torch.zeros(1, dtype=p.dtype, device=p.device), p.cumsum(0)[:-1]])
        p = p[before <= s["top_p"][r].double()]
        p = p / p.sum()
    at = int(torch.searchsorted(p.cumsum(0), s["uniforms"][r:r + 1].double(), right=True))
    return float(p[min(at, p.numel() - 1)].log())


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        rows = [_exact_row(s, r) for r in range(case["rows"])]
        return {"ids": None, "logprobs": torch.tensor(rows, dtype=torch.float64), "kept": None}
    if case["op"] == "clip":
        grads = [g.to(torch.float64) for g in s["grads"]]
        norm = math.sqrt(sum(float(torch.linalg.vector_norm(g)) ** 2 for g in grads))
        scale = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g.mul_(scale) for g in grads]}
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    z = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].detach().double())
    z.requires_grad_(case["train"])
    f = torch.nn.functional
    out = {"none": lambda t: t * 1.0, "relu": f.relu, "silu": f.silu, "gelu": f.gelu,
           "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[case["act"]](z)
    result = {"out": (out if s["residual"] is None else out + s["residual"].double()).detach()}
    if case["train"]:
        (dz,) = torch.autograd.grad(out, z, s["grad"].double())
        result.update(grad_x=torch.matmul(dz, w), grad_weight=torch.einsum("mn,mk->nk", dz, x))
        if s["bias"] is not None:
            result["grad_bias"] = torch.einsum("mn->n", dz)
        if s["residual"] is not None:
            result["grad_residual"] = s["grad"].double()
    return result
