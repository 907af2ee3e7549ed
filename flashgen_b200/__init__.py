"""flashgen_b200: B200-native (sm_100a) decode-step token sampler.

Drop-in for FlashGen's sampling path: ``SamplingParams`` and ``Sampler`` keep
the reference's call surface (flashgen/core/config.py, flashgen/sampling/
sampler.py) and run one fused CUDA kernel per call through the C ABI declared
in include/flashgen_sampler.h. Around the sampler: min-p; token log probabilities
with their gradient; a dense block and an LM head with per-request low-rank
adapters in front of it; gradient clipping for the step that trains them.
"""
from .core.config import SamplingParams  # noqa: F401
from .sampling.clip import clip_grad_norm, grad_norm  # noqa: F401
from .sampling.linear import HeadBlock, fused_linear  # noqa: F401
from .sampling.lm_head import AdapterHead  # noqa: F401
from .sampling.logprobs import (TokenLogprobs, logprobs_and_entropy, token_logprobs,  # noqa: F401
                                token_logprobs_grad)
from .sampling.min_p import MinPSample, sample_min_p  # noqa: F401
from .sampling.sampler import Sampler  # noqa: F401

__version__ = "0.1.0"
__all__ = ["SamplingParams", "Sampler", "AdapterHead", "TokenLogprobs", "token_logprobs", "token_logprobs_grad",
           "logprobs_and_entropy", "grad_norm", "clip_grad_norm", "fused_linear", "HeadBlock",
           "MinPSample", "sample_min_p"]
