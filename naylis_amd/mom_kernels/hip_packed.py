"""Causal attention over packed sequences (C ABI: naylis_mom_packed_attn_*).

The reference attends within batches of one length and equal heads
(model.py:279-345), which ``causal_attention`` does.  ``packed_attention`` is
the same read for sequences of different lengths laid end to end, as a prompt
pass or a packed training batch has them, with grouped heads, heads of 64 or
128, and keys of earlier tokens before a sequence's queries where there are any.
"""
from __future__ import annotations

from .. import _torch_ext


def packed_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, scale=None):
    """softmax(scale q k^T, causal within each sequence) v, differentiable.

    q (T, H, hd), k and v (Tk, Hkv, hd) bf16 with H a multiple of Hkv and hd 64
    or 128 (strided views are read in place where their rows are whole 16-byte
    pieces).  cu_seqlens (n + 1) int32 on the device: sequence i holds rows
    cu_seqlens[i] .. cu_seqlens[i + 1] - 1 of q; cu_seqlens_k likewise of k and
    v (default: the same).  The last query of a sequence sees its last key, each
    earlier one a key less; a query that sees none gives 0, and so do rows
    outside the sequences.  Offsets must not descend and are not copied to the
    host; they are clamped to the tensors.  scale defaults to hd ** -0.5.
    Returns (T, H, hd).  Scores may be of any size that fp32 holds.  Sequences do
    not see each other's rows, whatever these hold; within one, a weight of 0
    multiplies what it stands for as it is, so a NaN or an infinity reaches up to 62
    rows that have nothing to do with it: from a row of v the results, and of k or v
    the dq, of queries that see keys but not this one; from a row of dout the dv,
    and of q or dout the dk, of keys that its query does not see.  A forward with gradients keeps, beside its inputs and the output, what
    the output's rounding left (as much again) and (H, T) fp32.  The derivative of
    the backward and forward-mode derivatives raise."""
    return _torch_ext.load().packed_attention(q, k, v, cu_seqlens,
                                              cu_seqlens if cu_seqlens_k is None else cu_seqlens_k, scale, 0)
