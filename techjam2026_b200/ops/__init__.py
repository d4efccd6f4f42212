"""The CUDA kernels, re-exported with the reference's ops surface
(`kernelforge/ops/__init__.py:7-11`) plus the tcgen05 linear layer, the 8-bit
key/value cache and beam search's selection."""
from .layernorm import add_mask_layernorm, HAS_KERNELS
from .flash import flash_attention, flash_supported
from .gemm import linear, round_tf32
from .kv8 import (KV8Cache, kv8_append, kv8_attention, kv8_attention_shared, kv8_copy, kv8_evict,
                  kv8_read)
from .beam import beam_select

__all__ = ["add_mask_layernorm", "flash_attention", "flash_supported", "linear",
           "round_tf32", "HAS_KERNELS", "KV8Cache", "kv8_append", "kv8_attention",
           "kv8_attention_shared", "kv8_copy", "kv8_evict", "kv8_read", "beam_select"]
