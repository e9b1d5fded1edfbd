"""KV caches held in 4 bits: the size and shape of their pools.

A pool is one uint8 tensor (num_blocks, n_kv_heads, page_bytes) for K and V
together, a page being 16 tokens of one KV head.  Each 32 dims of a row share a
power-of-two scale, and a value takes 4 bits (a sign and one of 0, 0.5, 1, 1.5,
2, 3, 4, 6 times the scale): 136 bytes per token and KV head at head_dim 128,
where a bf16 cache holds 512.  include/femto_attn.h has the layout byte by byte.
The operators are ``femtovllm.ops.kv_cache_write_fp4`` and those named there.
"""

from __future__ import annotations

import torch

BLOCK_DIMS = 32


def page_bytes(head_dim: int) -> int:
    """Bytes of a page (16 tokens of K and V of one KV head)."""
    if head_dim <= 0 or head_dim > 128 or head_dim % 16:
        raise ValueError(f"head_dim must be at most 128 and a multiple of 16, got {head_dim}")
    return 512 * (-(-head_dim // BLOCK_DIMS)) + 128


def new_pool(num_blocks: int, n_kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A pool for one layer's K and V, zero-filled (every row reads as zeros)."""
    return torch.zeros((num_blocks, n_kv_heads, page_bytes(head_dim)), dtype=torch.uint8, device=device)
