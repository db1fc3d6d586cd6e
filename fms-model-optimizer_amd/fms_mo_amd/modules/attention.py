"""A paged key-value cache and the attention over it: what runs between a decoder layer's quantized q/k/v projection and its
output projection.  The reference keeps such a cache for its FP8 attention (fms_mo/aiu_addons/fp8/fp8_attn.py, whose products
are ``spyre::scaled_bmm``); there scores and probabilities pass through memory, here they do not leave the compute unit.
"""
from __future__ import annotations

import torch

from .. import kernels


class PagedKVCache:
    """Pages of keys and values of one layer.

    ``k``, ``v`` [pages, kv heads, page size, head dim] (a head's keys of a page lie together, so they are read as one piece); dtype
    float16, bfloat16, or float8_e4m3fn with one fp32 scale per key and head in ``k_scale`` / ``v_scale`` [pages, kv heads, page size].
    Which pages a sequence owns is the caller's: block_table int32 [B, pages of a sequence] (-1 where there is none), seq_lens
    int32 [B] counting the new tokens, query_start int32 [B + 1] where sequences have other than one new token."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
            raise TypeError(f"unsupported cache dtype {dtype}")
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        e4m3 = dtype == torch.float8_e4m3fn
        self.k_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device) if e4m3 else None
        self.v_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device) if e4m3 else None

    def store(self, q, k, v, block_table, seq_lens, query_start=None, **kw):
        """Normalize and rotate q and k, write k and v to their places, return q: ``kernels.qk_norm_rope_store``."""
        return kernels.qk_norm_rope_store(q, k, v, self.k, self.v, block_table, seq_lens, query_start, k_scale=self.k_scale,
                                          v_scale=self.v_scale, **kw)

    def attend(self, q, block_table, seq_lens, query_start=None, **kw):
        """Attention of the new tokens over what the cache holds of their sequences: ``kernels.paged_attention``."""
        return kernels.paged_attention(q, self.k, self.v, block_table, seq_lens, query_start, k_scale=self.k_scale,
                                       v_scale=self.v_scale, **kw)
