"""
Dropout whose mask is a function of a seed, an offset and the element's index: computed where it is applied, forward and
backward, and never stored.  The same seed and offset give the same mask on every call, whatever the type of the input, and in
whichever pieces of the GPU it is computed.

What is drawn: elements ``8g .. 8g+7`` (of the flat input, or of one frame of it) take the 16-bit halves, the lower one first,
of the four words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011), with the
seed as key and ``g`` and the offset as counter.  An element is dropped where its draw is below ``65536 * drop_prob``, rounded.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .sequence_lib import native

__all__ = ["dropout", "Dropout"]


def dropout(
    source: torch.Tensor,
    drop_prob: float,
    *,
    seed: int,
    offset: Union[int, torch.Tensor] = 0,
    residual: Optional[torch.Tensor] = None,
    same_over_time: bool = False,
) -> torch.Tensor:
    """
    :param source: any shape, float32 or bfloat16, on the GPU; time-major where ``same_over_time``.  (In a region of ``torch.autocast``
        float16 is taken as float32.)
    :param drop_prob: in [0,1], used as the nearest multiple of 1/65536, but neither 0 nor 1 where it is not; what is kept is scaled by
        ``1 / (1 - drop_prob)`` of that multiple
    :param seed: 64 bits
    :param offset: 64 bits, another one for every call that shall draw anew; or one int64 on the GPU, for calls that are recorded
        into a graph and draw anew at every replay.  (The gradient reads it again: change it after the backward pass.)
    :param residual: added to what comes out, in the same pass
    :param same_over_time: one mask for all frames, i.e. for all indices of axis 0
    :return: like ``source``; differentiable (once) with respect to ``source`` and ``residual``
    """
    drop_prob = float(drop_prob)
    if not 0.0 <= drop_prob <= 1.0:
        raise ValueError("dropout: drop_prob must be in [0,1], got %r" % drop_prob)
    threshold = int(round(drop_prob * 65536))
    if 0.0 < drop_prob < 1.0:
        threshold = min(max(threshold, 1), 65535)
    on_device = isinstance(offset, torch.Tensor)
    mask64 = (1 << 64) - 1
    return native().dropout(source, threshold, int(seed) & mask64, 0 if on_device else int(offset) & mask64, offset if on_device else None, residual, bool(same_over_time))


class Dropout(torch.nn.Module):
    """
    :func:`dropout` in training, nothing (but the residual's addition) in evaluation.  Every call in training takes the next
    offset; ``seed`` and ``offset`` are all the state there is, and setting them repeats the masks.  ``offset`` is in the
    ``state_dict``, so that a training that is taken up again goes on with the next masks.  (``seed`` is not: it belongs to the configuration, and
    ranks that train side by side on one saved state have seeds of their own.)
    """

    def __init__(self, drop_prob: float, *, seed: int = 0, same_over_time: bool = False):
        super().__init__()
        if not 0.0 <= float(drop_prob) <= 1.0:
            raise ValueError("Dropout: drop_prob must be in [0,1], got %r" % drop_prob)
        self.drop_prob, self.seed, self.same_over_time = float(drop_prob), int(seed), bool(same_over_time)
        self.offset = 0

    def forward(self, source: torch.Tensor, *, residual: Optional[torch.Tensor] = None, offset: Optional[Union[int, torch.Tensor]] = None) -> torch.Tensor:
        """
        :param residual: added to what comes out
        :param offset: of this call, as in :func:`dropout`, instead of the module's next one, which is left as it is.  A step that is recorded into a
            graph needs one on the GPU: the module's would be the same at every replay.  A segment that is recomputed in the backward pass
            (``torch.utils.checkpoint``) needs one as well: the module's next one is another than that of the first run.
        """
        if not self.training or self.drop_prob == 0.0:
            return source if residual is None else source + residual
        if residual is not None and residual.dtype != source.dtype:  # (as the addition in evaluation; a layer in an autocast region on a float32 input)
            both = torch.promote_types(source.dtype, residual.dtype)
            source, residual = source.to(both), residual.to(both)
        if offset is None:
            if source.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("%s: a recorded call would use one mask at every replay: give an offset on the GPU" % self)
            if torch._C._current_graph_task_id() != -1:  # (as torch.utils.checkpoint itself finds that it is in a backward pass)
                raise RuntimeError("%s: a call that is recomputed in a backward pass would take another mask than at first: give both an offset" % self)
            offset = self.offset
            self.offset += 1
        return dropout(source, self.drop_prob, seed=self.seed, offset=offset, residual=residual, same_over_time=self.same_over_time)

    def get_extra_state(self) -> torch.Tensor:
        """The offset, its 64 bits as an int64 (a tensor, as all else in a ``state_dict``)."""
        offset = int(self.offset) & ((1 << 64) - 1)
        return torch.tensor(offset - (1 << 64) if offset >> 63 else offset, dtype=torch.int64)

    def set_extra_state(self, state: torch.Tensor):
        self.offset = int(state) & ((1 << 64) - 1)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        missing_keys[:] = [k for k in missing_keys if k != prefix + "_extra_state"]  # (saved before there was one: the offset stays)

    def extra_repr(self) -> str:
        return "drop_prob=%g, seed=%i, same_over_time=%s" % (self.drop_prob, self.seed, self.same_over_time)
