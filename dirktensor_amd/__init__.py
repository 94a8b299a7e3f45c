"""dirktensor_amd — MI355X (gfx950) HIP implementation of DirkTensor's causal-attention path.

The kernels and the C ABI live in libdirktensor_amd.so (sources in csrc/,
declarations in include/dirktensor_amd.h); this package is the Python mirror
of the reference's FlashAttention.h / OlmoAttention.h interfaces on top of it.
"""

from .attention import (  # noqa: F401
    Context,
    FlashAttentionResult,
    OlmoAttention,
    default_context,
    flash_attention_backward,
    flash_attention_forward,
    qk_norm_rope,
)
from .cache import KVCache, cached_attention  # noqa: F401
from .drafts import VerifiedDrafts, verify_drafts  # noqa: F401
from .logprobs import TokenLogprobs, token_logprobs, token_logprobs_backward  # noqa: F401
from .model import OlmoModel, ce_loss  # noqa: F401
from .rotary import (  # noqa: F401
    HeadNormRotaryGradients,
    Rotary,
    head_norm_rotary,
    head_norm_rotary_backward,
    rotary,
    rotary_backward,
)
from ._workspace import release_workspaces  # noqa: F401
from ._capi import DTError, LIB_PATH  # noqa: F401

__all__ = [
    "Context",
    "DTError",
    "FlashAttentionResult",
    "HeadNormRotaryGradients",
    "KVCache",
    "LIB_PATH",
    "OlmoAttention",
    "OlmoModel",
    "Rotary",
    "TokenLogprobs",
    "VerifiedDrafts",
    "cached_attention",
    "ce_loss",
    "default_context",
    "flash_attention_backward",
    "flash_attention_forward",
    "head_norm_rotary",
    "head_norm_rotary_backward",
    "qk_norm_rope",
    "release_workspaces",
    "rotary",
    "rotary_backward",
    "token_logprobs",
    "token_logprobs_backward",
    "verify_drafts",
]
