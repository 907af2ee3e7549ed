"""The LM head over more rows than a decode batch has: a prompt scored under its adapters."""
import pytest
import torch

from tests.test_lm_head_gpu import DTYPES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,rank,slots", [(769, 8, 3), (1024, 16, 40), (1500, 48, 7), (2049, 16, 300), (5000, 128, 2)])
def test_many_rows(cuda_device, B, rank, slots, dtype):
    Case(B, 136, 300, rank, slots, dtype).check()
