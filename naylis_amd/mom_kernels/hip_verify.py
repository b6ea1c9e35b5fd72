"""Drafted tokens against a model's logits (C ABI: naylis_mom_verify_drafts).

The reference generates nothing (`use_cache=False`, pretrain.py:198).  Where a
serving loop drafts several tokens a step, appends them and reads the cache for
all of them at once (``paged_attention`` over N tokens), ``verify_drafts`` says
how many of them the model keeps and which token follows, from random numbers
that the caller draws.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _torch_ext


class VerifiedDrafts(NamedTuple):
    """tokens (B, N + 1) int64: the kept drafts, the token behind them, then -1;
    accepted (B,) int32, how many drafts were kept."""
    tokens: torch.Tensor
    accepted: torch.Tensor


def verify_drafts(logits, drafts, uniforms, draft_probs=None, draft_lens=None, temperature=1.0) -> VerifiedDrafts:
    """Keep each sequence's drafts as far as the model would have drawn them.

    logits (B, N + 1, V) bf16 or fp32: row i is the model's answer before draft
    drafts[b, i] (B, N), the last one behind all of them.  draft_probs (B, N, V)
    bf16 or fp32: the probabilities that the drafts were drawn from; without them
    the drafts came from a rule.  uniforms (B, N + 1) fp32 in [0, 1).  With p =
    softmax(logits / temperature): draft i is kept while uniforms[b, i] *
    draft_probs[b, i, draft] < p[b, i, draft]; the token behind the kept ones is
    the first whose cumulative weight exceeds uniforms[b, N] of the whole, in
    max(0, p - draft_probs) where a draft was turned away (without draft_probs: p
    without that draft), in p where none was.  So tokens are distributed as the
    model's own.

    draft_lens (B,) int32: drafts of each sequence (default N; clamped to [0, N]);
    the row behind them gives the token, later rows change nothing.  temperature: a
    number, finite and not negative, or (B,) fp32, where what is not above 0 counts as
    0 and infinity makes all columns but those of -inf alike; 0 takes the largest
    logit, the first of equal ones.  A column under 2 ** -900 of the likeliest one has
    no probability.  Columns of -inf have no probability; a row with a NaN, with +inf or with
    nothing else keeps no draft and gives token -1.  No backward."""
    temps = temperature if isinstance(temperature, torch.Tensor) else None
    tokens, accepted = _torch_ext.load().verify_drafts(logits, drafts, uniforms, draft_probs, draft_lens, temps,
                                                       1.0 if temps is not None else float(temperature), 0)
    return VerifiedDrafts(tokens, accepted)
