"""Forward-mode derivatives of the fused linear block are refused, not lost (no GPU: the refusal
comes before anything else)."""
import pytest
import torch
from torch.autograd import forward_ad

from flashgen_b200 import HeadBlock, fused_linear

BF16 = torch.bfloat16


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(which, grad):
    t = {"x": torch.zeros(3, 8, dtype=BF16), "weight": torch.zeros(8, 8, dtype=BF16), "bias": torch.zeros(8, dtype=BF16),
         "residual": torch.zeros(3, 8, dtype=BF16)}
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match=f"{which} carries a tangent"):
            fused_linear(**t)
        with pytest.raises(RuntimeError, match="carries a tangent"):
            HeadBlock(t["weight"], t["bias"])(t["x"]) if which != "residual" else fused_linear(**t)
        with pytest.raises(RuntimeError, match="GPU only"):     # no tangent: the next check
            fused_linear(**{k: torch.zeros(v.shape, dtype=BF16) for k, v in t.items()})
