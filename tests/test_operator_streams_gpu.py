"""The operators on streams and in captured graphs: behind a copy, a fill, a fork and join,
and behind each other, with every input rewritten between the runs."""
import pytest
import torch

from flashgen_b200 import AdapterHead, token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu


def _step(head, hidden, adapters, tokens, side):
    """Everything a call reads is written by the node just before it."""
    main = torch.cuda.current_stream()
    h = torch.empty_like(hidden)
    h.copy_(hidden)                                     # a copy, then the LM head
    logits = head.logits(h, adapters, out_dtype=torch.float32)
    first = token_logprobs(logits, tokens, top=5)       # behind a kernel
    fork = torch.cuda.Event()
    fork.record(main)
    side.wait_event(fork)
    with torch.cuda.stream(side):
        doubled = logits * 2
    join = torch.cuda.Event()
    join.record(side)
    main.wait_event(join)
    second = token_logprobs(doubled, tokens)            # behind a join
    weight = torch.empty(tokens.shape[0], device=hidden.device)
    weight.zero_()                                      # a fill, then the gradient
    zero = token_logprobs_grad(logits, tokens, first.max, first.logsum, weight)
    weight = weight + 1.5
    grad = token_logprobs_grad(logits, tokens, first.max, first.logsum, weight)
    again = token_logprobs(grad, tokens)
    return [logits, first.logprobs, first.entropy, first.rank, first.top_ids, first.top_logprobs, second.logprobs,
            second.entropy, zero, grad, again.logprobs, again.entropy]


def _inputs(batch, dim, vocab, slots, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(batch, dim, device="cuda", generator=g).to(torch.bfloat16)
    adapters = torch.randint(-1, slots, (batch,), device="cuda", generator=g, dtype=torch.int32)
    tokens = torch.randint(-1, vocab, (batch,), device="cuda", generator=g)
    return hidden, adapters, tokens


@pytest.mark.parametrize("batch,dim,vocab,rank", [(1, 64, 5000, 8), (7, 129, 1111, 16), (130, 256, 2500, 20)])
def test_graph_replays_match_eager_calls(batch, dim, vocab, rank):
    slots = 3
    head = AdapterHead(torch.randn(vocab, dim, device="cuda").to(torch.bfloat16) * dim ** -0.5, slots=slots, rank=rank)
    for s in range(slots):
        head.load(s, torch.randn(rank, dim, device="cuda") * dim ** -0.5, torch.randn(vocab, rank, device="cuda"), 0.5)
    static = _inputs(batch, dim, vocab, slots, 0)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        _step(head, *static, side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        out = _step(head, *static, side)
    for seed in (1, 2):
        fresh = _inputs(batch, dim, vocab, slots, seed)
        for t, f in zip(static, fresh):
            t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        with torch.cuda.stream(main):
            want = _step(head, *fresh, side)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_back_to_back_calls_read_finished_inputs():
    # each call's logits are the previous call's result: a kernel that began before its
    # predecessor's end would read the old ones
    vocab, batch = 70001, 64
    x = torch.randn(batch, vocab, device="cuda")
    tokens = torch.randint(0, vocab, (batch,), device="cuda")
    ones = torch.ones(batch, device="cuda")

    def chain(sync):
        y = x.clone()
        for _ in range(12):
            r = token_logprobs(y, tokens)
            if sync:
                torch.cuda.synchronize()
            token_logprobs_grad(y, tokens, r.max, r.logsum, ones, out=y)
            if sync:
                torch.cuda.synchronize()
            y.mul_(50.0)
            if sync:
                torch.cuda.synchronize()
        return y

    want = chain(True)
    for _ in range(3):
        assert torch.equal(chain(False), want)


@pytest.mark.parametrize("batch", [1, 40, 200])
@pytest.mark.parametrize("with_adapters", [False, True])
def test_the_head_reads_a_weight_written_just_before(batch, with_adapters):
    vocab, dim = 40003, 512
    versions = [torch.randn(vocab, dim, device="cuda").to(torch.bfloat16) * dim ** -0.5 for _ in range(4)]
    hidden = torch.randn(batch, dim, device="cuda").to(torch.bfloat16)
    weight = versions[0].clone()
    head = AdapterHead(weight, slots=2, rank=8)
    assert head.weight.data_ptr() == weight.data_ptr()
    head.load(1, torch.randn(8, dim, device="cuda"), torch.randn(vocab, 8, device="cuda"), 0.1)
    adapters = torch.arange(batch, device="cuda", dtype=torch.int32) % 3 - 1 if with_adapters else None

    def run(sync):
        out = []
        for v in versions:
            torch.mul(v, 1.0, out=weight)   # a kernel, not a copy
            if sync:
                torch.cuda.synchronize()
            out.append(head.logits(hidden, adapters))
            if sync:
                torch.cuda.synchronize()
        return out

    for got, want in zip(run(False), run(True)):
        assert torch.equal(got, want)
