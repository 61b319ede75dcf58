"""Scores of given tokens: log probability, entropy and the most probable alternatives of every row of logits, and the gradient of the
first two (csrc/logprobs.cuh, call site csrc/host_operators.cpp).  The reference's generation loop stops at the arg-max of the logits (generate.py:283, :305 of
Gu-J/TernaInfer); a program that scores texts, reports log probabilities or trains on them starts here."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .lib import load_host_call


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                    # fp32 [...], of the targets
    entropy: torch.Tensor                    # fp32 [...]
    top_logprob: Optional[torch.Tensor]      # fp32 [..., top]
    top_token: Optional[torch.Tensor]        # int64 [..., top]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """logits bf16, fp16 or fp32 [..., V] (V up to 2^19; up to 2^23 rows, any number of them where a row has at most 32 KB), targets int64 [...]:
    log softmax at the target (0 for a negative target, which stands for no token), entropy in nats, and with ``top`` (up to 32) the log
    probabilities and ids of the most probable tokens, the lowest id first among equal logits.  Logits of -inf (banned tokens) have probability
    0; a row without a finite logit gives NaN.  One pass over the logits; rows may be any distance apart.  Differentiable in the logits through
    ``logprob`` and ``entropy``.  A target of V or above gives NaN, as does a gradient other than 0 through it, and status 1 of the library."""
    return TokenLogprobs(*load_host_call().token_logprobs(logits, targets, top))
