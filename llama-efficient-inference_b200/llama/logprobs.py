"""What answers cost: log probabilities of given tokens, the entropy and the likeliest tokens (li4_token_logprobs).

The reference returns logits alone (llama/model.py:455-456); its sampling softmaxes and sorts all of them
(llama/generation.py:85-93).  Here one pass over a row of logits, in whatever type the projection left it, gives the numbers
that a user reads of it: Generation.generate_paged(logprobs=) returns them for the tokens it chose, Generation.score_paged
for the tokens of given texts.

Runs on the current stream of its tensors' device and allocates its outputs there; raises RuntimeError subclasses for
arguments it does not take.  No backward pass: tensors that require grad are refused outside torch.no_grad(); no registered
operator: fake tensors and calls under a tracer are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as native

MAX_TOP = 32  # LI4_MAX_TOP


class TokenLogprobs(NamedTuple):
    """Per row of logits; what was not asked for is None."""

    logprobs: Optional[torch.Tensor]      # fp32 [rows]: of the given tokens
    entropy: Optional[torch.Tensor]       # fp32 [rows], in nats
    top_tokens: Optional[torch.Tensor]    # int64 [rows, top]: the likeliest first, the lower index among equals
    top_logprobs: Optional[torch.Tensor]  # fp32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0,
                   entropy: bool = True) -> TokenLogprobs:
    """log softmax of each row of logits [rows, vocabulary] (float32, float16 or bfloat16, any row stride) at tokens
    int64 [rows], its entropy - sum p log p, and its `top` (0 to 32) likeliest tokens.

    Statistics in fp32.  A token outside the vocabulary gets NaN.  A logit of -infinity has probability 0 and adds 0 to the
    entropy; rows with a NaN or +infinity, or of nothing but -infinity, have NaN for their log probabilities and entropy,
    while their likeliest tokens are still in order (NaN above all)."""
    result = native.ext().token_logprobs(logits, tokens, top, entropy)
    if type(result) is int:
        native.check(result, "token_logprobs")
    return TokenLogprobs._make(result)
