"""DecodeBatch's rows over several requests: what a row's next request finds (CPU)."""
import torch

from flashgen_b200.core.config import SamplingParams
from flashgen_b200.sampling.decode import DecodeBatch


def test_a_reused_row_starts_its_sum_anew():
    dec = DecodeBatch([SamplingParams()] * 3, vocab=100, capacity=8, device="cpu")
    for r in range(3):
        dec.set_history(r, [1, 2, 3])
    assert dec.cumulative_logprob.tolist() == [0.0, 0.0, 0.0]
    dec.cumulative_logprob += torch.tensor([-1.5, -2.5, -3.5])         # steps of the first requests
    dec.set_history(1, [7])
    assert dec.cumulative_logprob.tolist() == [-1.5, 0.0, -3.5]
    assert dec.histories()[1] == [7]
