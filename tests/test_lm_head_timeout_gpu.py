"""A wait of the LM head's kernel that runs out: every row is marked, nothing is left unwritten, and the
next call is as ever. The products of one accumulator are computed and never reported
(fg_adapter_set_wait), so the wait for them ends at its limit of 5 ms."""
import pytest
import torch

from flashgen_b200 import SamplingParams, _lib
from flashgen_b200.sampling.decode import DecodeBatch
from tests.test_lm_head_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.fixture
def withheld():
    lib = _lib.load()

    def set_(accumulator):
        assert lib.fg_adapter_set_wait(5_000_000, accumulator) == _lib.FG_OK
    yield set_
    torch.cuda.synchronize()
    assert lib.fg_adapter_set_wait(0, -1) == _lib.FG_OK


# one CTA an accumulator and a pair, with adapters and without, sums in one piece and in several,
# one batch tile and three; the second tile of a CTA (or the second piece) is the one withheld, and the first
@pytest.mark.parametrize("accumulator", [0, 1])
@pytest.mark.parametrize("B,dim,V,dtype,out,adapters", [
    (1, 72, 40000, torch.bfloat16, torch.bfloat16, True), (40, 72, 40000, torch.float16, torch.float32, True),
    (40, 1100, 2000, torch.bfloat16, torch.float32, True), (70, 72, 40000, torch.float16, torch.float16, False),
    (200, 72, 80000, torch.bfloat16, torch.bfloat16, True), (200, 1100, 3000, torch.bfloat16, torch.float32, False),
    (700, 136, 30000, torch.float16, torch.float16, True)])
def test_a_wait_that_runs_out(cuda_device, withheld, B, dim, V, dtype, out, adapters, accumulator):
    c = Case(B, dim, V, 16, 3, dtype)
    ids = c.adapters if adapters else None
    want = c.exact(adapters=adapters).float().to(out)
    got = torch.full((B, V), 77.5, dtype=out, device="cuda")        # (an odd half: no exact result)
    withheld(accumulator)
    with pytest.raises(RuntimeError, match=f"pipeline timeout; {B} row"):
        c.head.logits(c.hidden, ids, out=got, check_errors=True)
    lost = got.isnan()
    assert lost.any(dim=1).all()                                    # some of every row
    assert (lost | (got == want)).all()                             # the rest is right, nothing is unwritten
    if accumulator == 1 and out != torch.float32 and B < 256:
        assert not lost.all()                                       # the first tiles came through
    withheld(-1)
    c.head.logits(c.hidden, ids, out=got, check_errors=True)
    assert torch.equal(got, want)


def test_a_step_whose_logits_did_not_come(cuda_device, withheld):
    """Without a check the sampler marks the rows: no id is drawn from what was not computed."""
    c = Case(9, 72, 40000, 16, 3, torch.bfloat16)
    dec = DecodeBatch([SamplingParams()] * 9, 40000, capacity=4)
    withheld(0)
    ids = dec.step_hidden(c.hidden, c.head, c.adapters, top_logprobs=1)
    assert (ids == -1).all() and (dec.cumulative_logprob == 0).all()
    strict = DecodeBatch([SamplingParams()] * 9, 40000, capacity=4, check_errors=True)
    with pytest.raises(RuntimeError, match="pipeline timeout"):
        strict.step_hidden(c.hidden, c.head, c.adapters)
    withheld(-1)
    assert (dec.step_hidden(c.hidden, c.head, c.adapters) >= 0).all()
