"""B200 CUDA kernels behind the reference's ``tritonforge.kernels`` API
(src/tritonforge/kernels/__init__.py:5-9), and the serving operators it does
not have: attention over packed prompts, the 4-bit KV cache and token log
probabilities."""

from __future__ import annotations

from .._lib import device_errors  # noqa: F401
from .dequant_gemm import quantized_linear  # noqa: F401
from .kv4 import (  # noqa: F401
    KV4Cache,
    kv4_decode_attention,
    kv4_decode_attention_rope,
    kv4_read,
    kv4_write,
    rope_kv4_write,
)
from .logprobs import token_logprobs  # noqa: F401
from .prompt_attention import prompt_attention  # noqa: F401
from .rmsnorm_residual import rmsnorm, rmsnorm_residual  # noqa: F401
from .swiglu import swiglu  # noqa: F401

__all__ = ["KV4Cache", "device_errors", "kv4_decode_attention", "kv4_decode_attention_rope", "kv4_read", "kv4_write",
           "prompt_attention", "quantized_linear", "rmsnorm", "rmsnorm_residual", "rope_kv4_write", "swiglu",
           "token_logprobs"]
