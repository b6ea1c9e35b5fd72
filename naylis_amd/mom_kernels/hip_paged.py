"""Paged key / value cache and the attention of a few new tokens over it (C ABI:
naylis_mom_paged_*).

The reference keeps no cache (`use_cache=False`, pretrain.py:198).  Here the
decoder's attention has what ``decode_step`` is for its MoM read: keys and
values of earlier tokens in pages, in bf16, as e4m3 codes with one fp32 scale
per token and head (the fp8 bank's form) or in 4 bits with a power of two per 32
features, filled by ``paged_append`` (``paged_append_rope`` rotates on the way)
and read by ``paged_attention``, or dense again by ``paged_gather``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _torch_ext

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class PagedCache(NamedTuple):
    """Pages k, v (pages, Hkv, page_size, head_dim), bf16, or uint8 e4m3 codes
    with k_scale, v_scale (pages, Hkv, page_size) fp32: k = k_scale * e4m3(k); or
    uint8 pairs of e2m1 codes (.., head_dim / 2), the even feature in the low four
    bits, with k_scale, v_scale (pages, Hkv, page_size, head_dim / 32) uint8: 32
    features times 2 ** (scale - 127), NaN for 255."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def dequantize(self):
        """(k, v) fp32: the values that the attention reads."""
        if self.k_scale is None:
            return self.k.float(), self.v.float()
        if self.k_scale.dtype == torch.uint8:
            return _e2m1_values(self.k, self.k_scale), _e2m1_values(self.v, self.v_scale)
        return (self.k.view(torch.float8_e4m3fn).float() * self.k_scale.unsqueeze(-1),
                self.v.view(torch.float8_e4m3fn).float() * self.v_scale.unsqueeze(-1))


def _e2m1_values(codes, scale):
    values = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), device=codes.device)
    x = values[torch.stack((codes & 15, codes >> 4), -1).long()].flatten(-2).unflatten(-1, (-1, 32))
    # 2 ** (scale - 127) from its bits (torch's pow is not exact on the GPU)
    bits = (scale.int() << 23).masked_fill(scale == 0, 1 << 22).masked_fill(scale == 255, 0x7fc00000)
    return (x * bits.view(torch.float32).unsqueeze(-1)).flatten(-2)


def new_paged_cache(pages, n_kv_heads, page_size, head_dim, device, fp8=False, fp4=False) -> PagedCache:
    """An empty cache; page_size a power of two in [16, 256], head_dim 64 or 128.
    fp8: e4m3 codes, fp4: e2m1 codes."""
    if fp8 and fp4:
        raise RuntimeError("new_paged_cache: fp8 and fp4 exclude each other")
    shape = (pages, n_kv_heads, page_size, head_dim)
    if fp4:
        return PagedCache(*(torch.zeros(*shape[:3], head_dim // 2, device=device, dtype=torch.uint8) for _ in range(2)),
                          *(torch.full((*shape[:3], head_dim // 32), 127, device=device, dtype=torch.uint8)
                            for _ in range(2)))
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


def paged_append_rope(cache: PagedCache, q, k, v, inv_freq, block_table, positions, rows=None, attention_scaling=1.0):
    """``paged_append`` with k rotated to its position on the way; returns q rotated.

    q (T, H, head_dim) bf16 (None: nothing is returned), the other arguments as
    there.  inv_freq (half,) fp32, half a multiple of 8 up to head_dim / 2: of each
    row's first 2 half features the pair (i, i + half) turns by the angle
    positions[t] * inv_freq[i], the others stay (transformers' rotation; the
    rotary embedding's inv_freq and attention_scaling are what it takes).
    Angles are formed in 64 bits, cosines and sines rounded to fp32 and results
    once, where ``rope`` takes them in the activations' type and keeps its
    roundings: in bf16 the two differ by those.  Tokens that are left out of the
    cache are rotated in q all the same.  No backward."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("paged_append_rope writes in place, which torch.jit.trace does not record")
    out = _torch_ext.load().paged_append_rope(*cache, q, k, v, inv_freq, block_table, positions, rows,
                                              float(attention_scaling), 0)
    return out if q is not None else None


def paged_gather(cache: PagedCache, block_table, cu_seqlens, tokens):
    """Sequences of the cache as dense rows (tokens, Hkv, head_dim) bf16: (k, v).

    Rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 are the first tokens of sequence
    b, whose pages block_table (B, W) names: what ``packed_attention`` takes, with
    cu_seqlens_k, for a prompt's chunk behind tokens of the cache.  cu_seqlens
    (B + 1) int32 stays on the device and must not descend; tokens is the number
    of rows to make.  Rows outside the sequences are 0, tokens past the table's
    row or in a page outside the cache NaN.  e4m3 values are rounded to bf16 with
    their scale, e2m1 values are exact (a value past bf16's largest is infinite).
    No backward."""
    k, v = _torch_ext.load().paged_gather(*cache, block_table, cu_seqlens, int(tokens), 0)
    return k, v


def paged_attention(q, cache: PagedCache, block_table, seq_lens, scale=None, q_lens=None):
    """Attention of one new token for each of B sequences over the cache, or of a few.

    q (B, H, head_dim) bf16, H a multiple of the cache's heads; block_table
    (B, W) and seq_lens (B,) int32.  Returns (B, H, head_dim) bf16: softmax(scale
    q k^T) v over the first seq_lens[b] tokens of sequence b (append the new
    token first), zeros for length 0, NaN for a length past the table's row or a
    page outside the cache.  scale defaults to head_dim ** -0.5.

    q (B, N, H, head_dim): N new tokens of each sequence (drafts behind the last
    token), all appended first; the last sees seq_lens[b] tokens, each earlier one
    a token less.  With q_lens (B,) int32 sequence b has the first q_lens[b] of
    its N rows (clamped to [0, N]), the last of those seeing all.  Rows behind
    them, and rows that see no token, are 0.  A new token weighs 0 in the rows
    that do not see it, so a NaN or an infinity in its v makes them NaN (one in
    its k does not).  No backward."""
    return _torch_ext.load().paged_attention(q, *cache, block_table, seq_lens, scale, q_lens, 0)
