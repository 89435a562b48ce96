"""
An embedding table: scaled rows of tokens, and the table's gradient, in which the errors of one token are added in the order of
their frames, by blocks of 8 to 32 of them, so that repeated calls agree bit for bit, whatever the other tokens are.
"""

from __future__ import annotations

from typing import Optional

import torch

from .model_lib import native

__all__ = ["embed", "Embedding"]


def embed(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """
    :param tokens: any shape, integers, on the GPU.  A negative one marks a frame without a token (padding): its row is 0, its error is not read.  One
        of V or more gives a row of NaN and adds nothing to the gradient.
    :param weight: [V,D] float32 or bfloat16, on the GPU; rows may have a pitch
    :param scale: of what comes out, e.g. the root of D
    :return: [...,D] in the type of ``weight``: ``scale * weight[token]``, differentiable (once) with respect to ``weight``; the gradient is dense,
        summed in float32
    """
    return native().embed(tokens, weight, float(scale))


class Embedding(torch.nn.Module):
    """:func:`embed` of a table of its own: ``weight [num_tokens, dim]``, initialised as that of ``torch.nn.Embedding`` (normal, standard deviation 1)."""

    def __init__(self, num_tokens: int, dim: int, *, scale: float = 1.0, device=None, dtype=None):
        super().__init__()
        self.num_tokens, self.dim, self.scale = int(num_tokens), int(dim), float(scale)
        self.weight = torch.nn.Parameter(torch.empty((self.num_tokens, self.dim), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self, generator: Optional[torch.Generator] = None):
        with torch.no_grad():
            self.weight.normal_(generator=generator)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embed(tokens, self.weight, scale=self.scale)

    def extra_repr(self) -> str:
        return "%i, %i, scale=%g" % (self.num_tokens, self.dim, self.scale)
