"""
A step of beam search: the best continuations over all hypotheses and tokens of each search, and the states of the hypotheses they go on from.
"""

from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import torch

from .model_lib import native

__all__ = ["beam_select", "reorder_states", "BeamStep"]


class BeamStep(NamedTuple):
    """Of each search the best first; ``...`` is the axis of the searches, if there is one."""

    totals: torch.Tensor  # [...,beam] float32
    sources: torch.Tensor  # [...,beam] int64: the hypotheses they go on from
    tokens: torch.Tensor  # [...,beam] int64


def beam_select(
    scores: torch.Tensor, totals: torch.Tensor, beam: int, *, ended: Optional[torch.Tensor] = None, end_token: Optional[int] = None
) -> BeamStep:
    """
    The ``beam`` largest of ``totals[b,k] + scores[b,k,v]`` (one addition in float32) of each search, in descending order, among equal ones the lowest
    hypothesis first and of one hypothesis the lowest token; a NaN before everything.

    :param scores: [B,K,V], or [K,V] of one search: log probabilities of the next token, of any model or sum of models, float32 or bfloat16, on the GPU; rows may
        have a pitch.  (In a region of ``torch.autocast`` float16 is taken as float32.)  The selection is not differentiable.
    :param totals: [B,K] or [K], float32, of the hypotheses so far; minus infinity for what is none (as all but one at a search's begin)
    :param beam: 1 to 64, at most K*V
    :param ended: [B,K] or [K] truth values: hypotheses that have ended go on with ``end_token`` and nothing else, at no cost, whatever their scores (which are not read)
    """
    return BeamStep(*native().beam_select(scores, totals, int(beam), ended, None if end_token is None else int(end_token)))


def reorder_states(states: Sequence[torch.Tensor], sources: torch.Tensor) -> List[torch.Tensor]:
    """
    :param states: tensors [B,K,...] of any types, or [K,...] of one search, on the GPU
    :param sources: [B,beam] or [beam] int64, as of :class:`BeamStep`
    :return: the rows of the sources, [B,beam,...] or [beam,...]; zeros where a source is not in 0..K-1.  Not differentiable.
    """
    return native().reorder_states(list(states), sources)
