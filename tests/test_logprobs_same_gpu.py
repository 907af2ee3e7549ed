"""The same id has the same log probability, bit for bit, as the token and as an alternative."""
import pytest
import torch

from flashgen_b200.sampling.logprobs import token_logprobs
from tests.test_logprobs_gpu import DTYPES, _random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", [(1, 50257), (6, 1000), (150, 9001), (500, 3000)])
def test_token_and_alternative_agree(cuda_device, B, V, dtype):
    x, _, T = _random(B, V, dtype, V)
    ids = token_logprobs(x, top=32).top_ids
    for temperature in (T, T * 37.3, None):
        for place in (0, 1, 7, 31):
            r = token_logprobs(x, ids[:, place].contiguous(), temperature=temperature, top=32)
            assert torch.equal(r.top_ids, ids)
            assert (r.rank == place).all()
            assert torch.equal(r.logprobs, r.top_logprobs[:, place])
