"""Log probabilities of tokens under their logits (C ABI: naylis_mom_logprobs_*).

The reference keeps the summed loss of such rows (model.py:536-545), which
``cross_entropy_rows`` computes.  ``token_logprobs`` is what scoring, sampling
reports and policy gradients need of them: each token's log probability, the
row's entropy and its likeliest tokens, in one pass over the logits.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _torch_ext


class TokenLogprobs(NamedTuple):
    """logp and entropy (...) fp32, differentiable; top_ids (..., top) int64 and
    top_logp (..., top) fp32, without gradient, None for top = 0."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logp: Optional[torch.Tensor]


def token_logprobs(logits, tokens, top=0, ignore_index=-100) -> TokenLogprobs:
    """Log probability of tokens (...) under bf16 or fp32 logits (..., V).

    logp is 0 (with no gradient) where the token is ignore_index, NaN where it
    is neither that nor in [0, V).  Columns of -inf have no probability and add
    nothing; finite logits may be of any size.  top (up to 64) gives each row's
    largest logits, equal ones by the lowest index.  The derivative of
    the backward and forward-mode derivatives raise."""
    logp, entropy, ids, lps = _torch_ext.load().token_logprobs(logits, tokens, int(top), int(ignore_index), 0)
    return TokenLogprobs(logp, entropy, ids if top else None, lps if top else None)
