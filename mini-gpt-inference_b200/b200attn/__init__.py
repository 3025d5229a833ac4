"""b200attn -- sm_100a paged-attention backend for the minivllm runtime.

Public API (CUDA only, no fallback):
  paged_attention_batch_b200  -- batched paged decode attention (+ fused KV write)
  kv_scatter_b200             -- slot-mapping KV-cache scatter
  chunked_prefill_b200        -- prefix-aware chunked-prefill attention
  chunked_prefill_batch_b200  -- several prefill chunks in one launch
  qkv_kv_write_b200           -- QKV projection with the KV write in its epilogue (bf16)
  qk_norm_rope_b200           -- RMS norm of each q/k head and position rotation, in one pass
  rope_kv_append_b200         -- the same, with k and v appended to the paged pool
  rope_table                  -- the table of cosines and sines that the two read
  shared_prefix_decode_b200   -- paged decode of a batch that shares a prefix, read once
  selftest_bounded_wait       -- device check of the kernels' bounded-wait error path
Importing the package also registers torch.ops.b200attn.{paged_decode,
kv_scatter, chunked_prefill, qkv_kv_write, qk_norm_rope, rope_kv_append,
shared_prefix_decode} (see torch_ops.py).
"""
from .ops import (chunked_prefill_b200, chunked_prefill_batch_b200, decode_bytes,
                  is_available, kv_scatter_b200, paged_attention_batch_b200,
                  qkv_kv_write_b200, selftest_bounded_wait)
from .rope import qk_norm_rope_b200, rope_kv_append_b200, rope_table
from .shared_prefix import shared_prefix_decode_b200
from ._lib import LIB_PATH, load as load_library
from . import torch_ops  # registers torch.ops.b200attn.*

__all__ = [
    "paged_attention_batch_b200", "kv_scatter_b200", "chunked_prefill_b200",
    "chunked_prefill_batch_b200", "qkv_kv_write_b200", "selftest_bounded_wait", "decode_bytes", "is_available",
    "qk_norm_rope_b200", "rope_kv_append_b200", "rope_table", "shared_prefix_decode_b200",
    "load_library", "LIB_PATH",
]
