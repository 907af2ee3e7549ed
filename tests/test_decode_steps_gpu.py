"""DecodeBatch's steps that fail, and what they leave behind."""
import pytest
import torch

from flashgen_b200 import SamplingParams
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
