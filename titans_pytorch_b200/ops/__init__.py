"""Operators: each runs an sm_100a kernel on CUDA tensors and a PyTorch restatement on CPU."""

from ._ext import available as kernels_available
from ._ext import want_kernels
from .attention import window_attention
from .conv import conv_silu_norm
from .decode_attention import decode_attention
from .ffn import swiglu_ffn
from .kv_cache import KVCache, kv_cache_read, kv_cache_write
from .memory import memory_step
from .norm import rms_norm
from .rope import rope_frequencies, rotary_embedding
from .sampling import sample_tokens

__all__ = ["kernels_available", "want_kernels", "window_attention", "conv_silu_norm",
           "swiglu_ffn", "memory_step", "rms_norm", "rope_frequencies", "rotary_embedding", "KVCache",
           "kv_cache_write", "kv_cache_read", "decode_attention", "sample_tokens"]
