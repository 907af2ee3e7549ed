"""DecodeBatch's steps that fail, and what they leave behind."""
import pytest
import torch

from flashgen_b200 import AdapterHead, SamplingParams
from flashgen_b200.sampling.decode import DecodeBatch

pytestmark = pytest.mark.gpu


def test_a_failed_step_leaves_no_log_probabilities(cuda_device):
    dec = DecodeBatch([SamplingParams()] * 3, 500, capacity=8, check_errors=True)
    logits = torch.randn(3, 500, device="cuda")
    dec.step(logits, top_logprobs=2)
    assert dec.last_logprobs is not None
    kept = dec.cumulative_logprob.clone()
    logits[1] = float("nan")
    with pytest.raises(RuntimeError, match="nan"):
        dec.step(logits, top_logprobs=2)
    assert dec.last_logprobs is None
    assert torch.equal(dec.cumulative_logprob, kept)
    assert [len(h) for h in dec.histories()] == [1, 1, 1]
    with pytest.raises(AssertionError):
        dec.step(logits[:2], top_logprobs=2)
    assert dec.last_logprobs is None


def _head(V=500, dim=64, slots=2):
    head = AdapterHead(torch.randn(V, dim, device="cuda").half() * dim ** -0.5, slots=slots, rank=8)
    for i in range(slots):
        head.load(i, torch.randn(8, dim, device="cuda") * dim ** -0.5, torch.randn(V, 8, device="cuda"))
    return head


def test_bad_adapters_raise_where_errors_are_checked(cuda_device):
    head = _head()
    hidden = torch.randn(3, 64, device="cuda").half()
    bad = torch.tensor([0, 5, -1], dtype=torch.int32, device="cuda")
    dec = DecodeBatch([SamplingParams()] * 3, 500, capacity=8, check_errors=True)
    dec.step_hidden(hidden, head, bad.clamp(max=1), top_logprobs=1)
    with pytest.raises(RuntimeError, match="row 1"):
        dec.step_hidden(hidden, head, bad, top_logprobs=1)
    assert dec.last_logprobs is None and [len(h) for h in dec.histories()] == [1, 1, 1]
    ids = DecodeBatch([SamplingParams()] * 3, 500, capacity=8).step_hidden(hidden, head, bad)   # not checked: shared logits
    assert (ids >= 0).all()


@pytest.mark.parametrize("out_dtype", [None, torch.float16, torch.float32])
def test_logits_of_a_step_from_hidden_states(cuda_device, out_dtype):
    head = _head()
    hidden = torch.randn(3, 64, device="cuda").half()
    ad = torch.tensor([0, 1, -1], dtype=torch.int32, device="cuda")
    u = torch.full((3,), 0.3, device="cuda")
    a, b = (DecodeBatch([SamplingParams()] * 3, 500, capacity=8) for _ in range(2))
    ids = a.step_hidden(hidden, head, ad, out_dtype=out_dtype, uniforms=u, top_logprobs=3)
    assert torch.equal(ids, b.step(head.logits(hidden, ad, out_dtype=out_dtype), uniforms=u, top_logprobs=3))
    for x, y in zip(a.last_logprobs, b.last_logprobs):
        assert torch.equal(x, y)
    with pytest.raises(TypeError):
        a.step_hidden(hidden, head, ad, out_dtype=torch.bfloat16)
