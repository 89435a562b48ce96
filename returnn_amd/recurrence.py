"""
A gated linear recurrence: a recurrent layer that is parallel in time.

:func:`gated_recurrence` is ``NativeLstm2`` without its recurrent product (returnn/native_op.py:1029-1121: the same gates in the
same order, the same masking of frames past a sequence's end, the same carrying of the state), so that the state follows
a recurrence that is linear in it and can be computed for many frames at once::

    c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(z_t),    y_t = sigmoid(o_t) c_t

(ifo pooling of Bradbury, Merity, Xiong, Socher: Quasi-recurrent neural networks, 2016.)  :class:`GatedRecurrence` is the layer
on top of it, the counterpart of :class:`returnn_amd.lstm.LSTM`: projection, recurrence, and one step for search.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from .sequence_lib import native

__all__ = ["gated_recurrence", "GatedRecurrence"]


def gated_recurrence(
    source: torch.Tensor, *, state: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None, direction: int = 1
) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    :param source: [T,B,4*out] gates before their activation, time-major, or [B,4*out] for a single step; along the last axis
        cell-in, input, forget, output; float32 or bfloat16, on the GPU; rows may have a pitch (e.g. a slice of a wider projection).  (In a
        region of ``torch.autocast`` float16, which a projection gives there, is taken as float32.)
    :param state: [B,out] before the first frame, default zeros
    :param seq_lens: [B] integer lengths (any device), None = all sequences have T frames.  Frames past them are not read, their
        output is 0 and they leave the state as it is.
    :param direction: +1, or -1 to go from each sequence's last frame to its first
    :return: output [T,B,out] (or [B,out]) in the type of ``source``, state [B,out] after the last frame visited, float32.
        Both differentiable (once) with respect to ``source`` and ``state``.
    """
    return native().gated_recurrence(source, state, seq_lens, direction)


class GatedRecurrence(torch.nn.Module):
    """
    Projection and gated linear recurrence.  Parameters ``ff [4*out, in]`` and ``bias [4*out]``, gate blocks in the order
    cell-in, input, forget, output.  Initialisation: ``ff`` Glorot-uniform (returnn/frontend/init.py:189-197), ``bias`` zero but
    for the forget gates, which start at ``forget_bias``: at 0 a state would be gone after a few frames.
    """

    def __init__(self, in_dim: int, out_dim: int, *, forget_bias: float = 2.0, device=None, dtype=None):
        super().__init__()
        self.in_dim, self.out_dim, self.forget_bias = int(in_dim), int(out_dim), float(forget_bias)
        kw = dict(device=device, dtype=dtype)
        self.ff = torch.nn.Parameter(torch.empty((4 * self.out_dim, self.in_dim), **kw))
        self.bias = torch.nn.Parameter(torch.empty((4 * self.out_dim,), **kw))
        self.reset_parameters()

    def reset_parameters(self, generator: Optional[torch.Generator] = None):
        n = self.out_dim
        with torch.no_grad():
            limit = math.sqrt(6.0 / (n + self.in_dim))  # (each gate is a layer of its own)
            self.ff.uniform_(-limit, limit, generator=generator)
            self.bias.zero_()
            self.bias[2 * n : 3 * n] = self.forget_bias

    def forward(
        self, source: torch.Tensor, *, state: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None, direction: int = 1
    ) -> Tuple[torch.Tensor, torch.Tensor]:
        """
        :param source: [T,B,in], or [B,in] for a single step
        :param state: [B,out] or None (zeros)
        :param seq_lens: [B] or None
        :return: output [T,B,out] (or [B,out]), new state [B,out].  As for the LSTM layer the projection runs in an autocast region's type, and
            the output is bfloat16 where that is, else float32.
        """
        if source.shape[-1] != self.in_dim:
            raise ValueError("%s: input %s does not have in_dim %i" % (self, tuple(source.shape), self.in_dim))
        gates = torch.nn.functional.linear(source, self.ff, self.bias)
        return gated_recurrence(gates, state=state, seq_lens=seq_lens, direction=direction)

    def default_initial_state(self, *, batch_dims: Sequence[int], device=None) -> torch.Tensor:
        """zeros, float32"""
        return torch.zeros(tuple(batch_dims) + (self.out_dim,), dtype=torch.float32, device=device or self.ff.device)

    def extra_repr(self) -> str:
        return "in_dim=%i, out_dim=%i" % (self.in_dim, self.out_dim)
