"""Sampling with penalties while no row has a history yet."""
import pytest
import torch

from flashgen_b200 import Sampler, SamplingParams

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("min_p", [0.0, 0.1])
@pytest.mark.parametrize("batch", [1, 3, 300])
def test_empty_histories(cuda_device, min_p, batch):
    x = torch.randn(batch, 5000, device="cuda")
    u = torch.rand(batch, device="cuda")
    p = [SamplingParams(repetition_penalty=1.3, min_p=min_p)] * batch
    want = Sampler().sample(x, p, uniforms=u)
    offsets = torch.zeros(batch + 1, dtype=torch.int64)
    for history in ([[] for _ in range(batch)], (torch.zeros(0, dtype=torch.int32), offsets),
                    (torch.zeros(0, dtype=torch.int32), offsets, 0)):
        assert torch.equal(Sampler().sample(x, p, token_histories=history, uniforms=u), want)
