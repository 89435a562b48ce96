"""
What comes behind the output projection of a language model or decoder: log probabilities of given tokens, the entropy of the
distribution, and the best alternatives, in one pass over the logits; and their gradient, in one more.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .sequence_lib import native

__all__ = ["token_log_probs", "TokenScores"]


class TokenScores(NamedTuple):
    """All but ``top_ids`` float32; ``...`` are the axes of the logits but the last."""

    log_probs: Optional[torch.Tensor]  # [...] of the targets, None without targets
    entropy: Optional[torch.Tensor]  # [...], in nats, None if not asked for
    top_log_probs: torch.Tensor  # [...,top_k] in descending order
    top_ids: torch.Tensor  # [...,top_k] int64


def token_log_probs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, entropy: bool = False, top_k: int = 0) -> TokenScores:
    """
    :param logits: [...,V] float32 or bfloat16, on the GPU; rows may have a pitch (e.g. those of a vocabulary padded in the projection).
        A logit of minus infinity is a token that is not allowed: probability 0.  (In a region of ``torch.autocast`` float16 is taken as float32.)
    :param targets: [...] integer tokens, or None.  A negative one marks a row without a token (padding): it is not read, its
        log probability, entropy and gradient are 0, its alternatives have log probability minus infinity and index -1.
        One of V or more makes its log probability and the gradient of its row NaN.
    :param entropy: whether it is wanted
    :param top_k: how many alternatives, 0 to 64: the largest logits, among equal ones the lower index first
    :return: log probabilities and entropy are differentiable (once) with respect to the logits, the alternatives are not.  A row in which
        no token is allowed has log probabilities of minus infinity, entropy 0 and gradient 0.
    """
    return TokenScores(*native().token_log_probs(logits, targets, bool(entropy), int(top_k)))
