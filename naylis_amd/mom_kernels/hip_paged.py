"""Paged key / value cache and the attention of one new token over it (C ABI:
naylis_mom_paged_*).

The reference keeps no cache (`use_cache=False`, pretrain.py:198).  Here the
decoder's attention has what ``decode_step`` is for its MoM read: keys and
values of earlier tokens in pages, in bf16 or as e4m3 codes with one fp32 scale
per token and head (the fp8 bank's form), filled by ``paged_append`` and read
by ``paged_attention``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _torch_ext


class PagedCache(NamedTuple):
    """Pages k, v (pages, Hkv, page_size, head_dim), bf16, or uint8 e4m3 codes
    with k_scale, v_scale (pages, Hkv, page_size) fp32: k = k_scale * e4m3(k)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def dequantize(self):
        """(k, v) fp32: the values that the attention reads."""
        if self.k_scale is None:
            return self.k.float(), self.v.float()
        return (self.k.view(torch.float8_e4m3fn).float() * self.k_scale.unsqueeze(-1),
                self.v.view(torch.float8_e4m3fn).float() * self.v_scale.unsqueeze(-1))


def new_paged_cache(pages, n_kv_heads, page_size, head_dim, device, fp8=False) -> PagedCache:
    """An empty cache; page_size a power of two in [16, 256], head_dim 64 or 128."""
    shape = (pages, n_kv_heads, page_size, head_dim)
    dtype = torch.uint8 if fp8 else torch.bfloat16
    k, v = (torch.zeros(shape, device=device, dtype=dtype) for _ in range(2))
    if not fp8:
        return PagedCache(k, v)
    return PagedCache(k, v, *(torch.ones(shape[:3], device=device) for _ in range(2)))


def paged_append(cache: PagedCache, k, v, block_table, positions, rows=None):
    """Write new tokens' k, v (T, Hkv, head_dim) bf16 into the cache, in place.

    block_table (B, W) int32: each sequence's pages in order.  Token t becomes
    token positions[t] of sequence rows[t]; without rows, of sequence t.  Tokens
    whose position, row or page is outside the table or the cache (position -1
    for padding) are left out.  No two tokens of a call may have the same place.
    No backward: raises where k or v want a gradient."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("paged_append writes in place, which torch.jit.trace does not record")
    _torch_ext.load().paged_append(*cache, k, v, block_table, positions, rows, 0)


def paged_attention(q, cache: PagedCache, block_table, seq_lens, scale=None):
    """Attention of one new token for each of B sequences over the cache.

    q (B, H, head_dim) bf16, H a multiple of the cache's heads; block_table
    (B, W) and seq_lens (B,) int32.  Returns (B, H, head_dim) bf16: softmax(scale
    q k^T) v over the first seq_lens[b] tokens of sequence b (append the new
    token first), zeros for length 0, NaN for a length past the table's row or a
    page outside the cache.  scale defaults to head_dim ** -0.5.  No backward."""
    return _torch_ext.load().paged_attention(q, *cache, block_table, seq_lens, scale, 0)
