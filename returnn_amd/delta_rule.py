"""
The gated delta rule: a recurrent layer whose state is a matrix per head, which learns to answer keys with values and to forget.

:func:`gated_delta_rule` computes, for every head, with ``a_t = exp(log_decay_t)``::

    S_t = a_t S_{t-1} + k_t u_t^T,    u_t = beta_t (v_t - a_t S_{t-1}^T k_t),    y_t = scale S_t^T q_t

(Yang, Kautz, Hatamizadeh: Gated delta networks: improving Mamba2 with delta rule, 2024.)  Frames past a sequence's end give 0 and leave the state, as in
:func:`returnn_amd.recurrence.gated_recurrence`.  :class:`DeltaRecurrence` is the layer on top of it.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from .model_lib import native

__all__ = ["gated_delta_rule", "DeltaRecurrence"]


def gated_delta_rule(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    *,
    scale: Optional[float] = None,
    state: Optional[torch.Tensor] = None,
    seq_lens: Optional[torch.Tensor] = None,
    direction: int = 1,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    :param query: [T,B,key_heads,dk], time-major, or [B,key_heads,dk] for a single step; float32 or bfloat16, on the GPU; 1 <= dk <= 128; frames may have a pitch
        (e.g. a slice of a wider projection), of all sequences together up to 64 MiB.  (In a region of ``torch.autocast`` float16 is taken as float32.)
    :param key: like ``query``.  A step multiplies what the state holds along the key by ``exp(log_decay) (1 - beta |key|^2)``: with ``beta |key|^2`` above 2 it grows without bounds unless
        it decays.  (With ``beta`` near 2 keys have to be a little shorter than 1: rounded to bfloat16, keys of length 1 can be longer by 2^-8.)
    :param value: [T,B,heads,dv] or [B,heads,dv] of the same type; ``heads`` is a multiple of ``key_heads``, neighbouring heads share queries and keys
    :param log_decay: [T,B,heads] or [B,heads], at most 0, taken as float32; minus infinity forgets all that was before
    :param beta: like ``log_decay``; how much of what is missing is written, 0 to 1 (up to 2 for states that may change their sign)
    :param scale: of the output, default ``dk ** -0.5``
    :param state: [B,heads,dk,dv] before the first frame, default zeros
    :param seq_lens: [B] integer lengths (any device), None = all sequences have T frames.  Frames past them are not read, their output is 0 and they leave
        the state as it is.
    :param direction: +1, or -1 to go from each sequence's last frame to its first
    :return: output like ``value``, state [B,heads,dk,dv] after the last frame visited, float32.
        Both differentiable (once) with respect to all inputs but the lengths.  A number that is not finite (or, of a float32 state or value, above 3.38e38, the largest of bfloat16)
        spoils the outputs of its head from the 64 frames (float32: 32) that are computed with it on, not from its own frame on; in a call of up to 16 frames without a gradient, from its own.
    """
    return native().gated_delta_rule(query, key, value, log_decay, beta, scale, state, seq_lens, direction)


class DeltaRecurrence(torch.nn.Module):
    """
    Projection and gated delta rule, the counterpart of :class:`returnn_amd.recurrence.GatedRecurrence`.  Parameters ``ff`` and ``bias`` of
    queries ``[num_heads*key_dim]``, keys (the same), values ``[out_dim]``, decays and betas ``[num_heads]`` each, in this order.  Queries and keys are brought to
    length 1, ``log_decay = -softplus``, ``beta = sigmoid``.  Initialisation: ``ff`` Glorot-uniform, ``bias`` zero but for the decays, which start at ``decay_bias``.

    :param num_heads: divides out_dim; default: heads of 64, or one
    :param key_dim: of a head, up to 128; default: that of its values, at most 128
    """

    def __init__(
        self, in_dim: int, out_dim: int, *, num_heads: Optional[int] = None, key_dim: Optional[int] = None, decay_bias: float = -3.0, device=None, dtype=None
    ):
        super().__init__()
        self.in_dim, self.out_dim, self.decay_bias = int(in_dim), int(out_dim), float(decay_bias)
        self.num_heads = int(num_heads) if num_heads is not None else (self.out_dim // 64 if self.out_dim % 64 == 0 and self.out_dim else 1)
        if self.num_heads < 1 or self.out_dim % self.num_heads:
            raise ValueError("DeltaRecurrence: %i heads cannot share %i channels evenly" % (self.num_heads, self.out_dim))
        self.value_dim = self.out_dim // self.num_heads
        self.key_dim = int(key_dim) if key_dim is not None else min(self.value_dim, 128)
        if not 1 <= self.key_dim <= 128:
            raise ValueError("DeltaRecurrence: key_dim must be 1 to 128, got %i" % self.key_dim)
        self.split = [self.num_heads * self.key_dim] * 2 + [self.out_dim] + [self.num_heads] * 2
        kw = dict(device=device, dtype=dtype)
        self.ff = torch.nn.Parameter(torch.empty((sum(self.split), self.in_dim), **kw))
        self.bias = torch.nn.Parameter(torch.empty((sum(self.split),), **kw))
        self.reset_parameters()

    def reset_parameters(self, generator: Optional[torch.Generator] = None):
        with torch.no_grad():
            for w in self.ff.split(self.split):  # (each a layer of its own)
                limit = (6.0 / (w.shape[0] + self.in_dim)) ** 0.5
                w.uniform_(-limit, limit, generator=generator)
            self.bias.zero_()
            self.bias.split(self.split)[3].fill_(self.decay_bias)

    def forward(
        self, source: torch.Tensor, *, state: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None, direction: int = 1
    ) -> Tuple[torch.Tensor, torch.Tensor]:
        """
        :param source: [T,B,in], or [B,in] for a single step
        :param state: [B,num_heads,key_dim,out/num_heads] or None (zeros)
        :param seq_lens: [B] or None
        :return: output [T,B,out] (or [B,out]), new state.  As for the other layers the projection runs in an autocast region's type, and the output is
            bfloat16 where that is, else float32.
        """
        if source.shape[-1] != self.in_dim:
            raise ValueError("%s: input %s does not have in_dim %i" % (self, tuple(source.shape), self.in_dim))
        q, k, v, g, b = torch.nn.functional.linear(source, self.ff, self.bias).split(self.split, dim=-1)
        q, k = (self._unit(t.unflatten(-1, (self.num_heads, self.key_dim))) for t in (q, k))
        v = v.unflatten(-1, (self.num_heads, self.value_dim))
        y, s = gated_delta_rule(
            q, k, v, -torch.nn.functional.softplus(g.float()), torch.sigmoid(b.float()), state=state, seq_lens=seq_lens, direction=direction
        )
        return y.flatten(-2), s

    @staticmethod
    def _unit(t: torch.Tensor) -> torch.Tensor:
        x = t.float()
        return (x * torch.rsqrt(x.square().sum(dim=-1, keepdim=True) + 1e-6)).to(t.dtype)

    def default_initial_state(self, *, batch_dims: Sequence[int], device=None) -> torch.Tensor:
        """zeros, float32"""
        return torch.zeros(tuple(batch_dims) + (self.num_heads, self.key_dim, self.value_dim), dtype=torch.float32, device=device or self.ff.device)

    def extra_repr(self) -> str:
        return "in_dim=%i, out_dim=%i, num_heads=%i, key_dim=%i" % (self.in_dim, self.out_dim, self.num_heads, self.key_dim)
