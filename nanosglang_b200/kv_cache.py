"""An 8-bit key/value cache: one layer's pages, written, read back and attended over.

The reference keeps keys and values in the model's 16-bit dtype in pages of
``[blocks, block_size, kv_heads, head_dim]`` per layer
(nano_sglang/engine/paged_kv_cache.py:62-69). This cache holds the same pages
as int8 or e4m3 codes with one fp32 scale per token and kv head: about half the
memory, and half the bytes that a decode step reads.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops

__all__ = ["QuantizedKVCache"]

_CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


class QuantizedKVCache:
    """Pages of 8-bit keys and values of one layer.

    ``k``, ``v``: codes [pages, page_size, kv_heads, head_dim]; ``k_scale``,
    ``v_scale``: float32 [pages, page_size, kv_heads]. They are views of
    head-major memory (a head's tokens of a page are contiguous, which is how
    decode attention reads them). A token's place is the slot ``page *
    page_size + offset``. Pages of a multiple of 16 tokens take the faster
    attention path. The caller owns the page tables and the lengths; every call
    is stream-ordered and can be captured in a CUDA graph.
    """

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, codes: str = "int8", device=None):
        if codes not in _CODES:
            raise ValueError(f"codes must be one of {sorted(_CODES)}, got {codes!r}")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 16 from 16 to 256, got {head_dim}")
        shape = (pages, kv_heads, page_size)

        def pool():
            c = torch.zeros(*shape, head_dim, dtype=torch.int8, device=device).view(_CODES[codes])
            return c.transpose(1, 2), torch.zeros(shape, dtype=torch.float32, device=device).transpose(1, 2)

        self.k, self.k_scale = pool()
        self.v, self.v_scale = pool()
        self.page_size = page_size

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise k, v [T, kv_heads, head_dim] into ``slots`` (int64 [T]): ``ops.kv_cache_write``."""
        ops.kv_cache_write(k, v, self.k, self.v, self.k_scale, self.v_scale, slots)

    def read(self, slots: torch.Tensor, dtype: torch.dtype):
        """(k, v) [T, kv_heads, head_dim] at ``slots``: ``ops.kv_cache_read``."""
        return ops.kv_cache_read(self.k, self.v, self.k_scale, self.v_scale, slots, dtype)

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
               softmax_scale: Optional[float] = None, return_lse: bool = False):
        """Attention of one query token per sequence: ``ops.kv_attention_decode``."""
        return ops.kv_attention_decode(q, self.k, self.v, self.k_scale, self.v_scale, page_table, seq_lens,
                                       softmax_scale, return_lse)
