"""
A recurrent language model of this package's operators: the path on which they run together.

Embedding (:class:`returnn_amd.embedding.Embedding`), a stack of recurrent layers (:class:`returnn_amd.recurrence.GatedRecurrence`,
:class:`returnn_amd.delta_rule.DeltaRecurrence` or :class:`returnn_amd.lstm.LSTM`) with dropout between them, added to what went in, and a projection to
the vocabulary, whose logits go through :func:`returnn_amd.scoring.token_log_probs`: the loss in training, scores of given texts, and the alternatives of
every hypothesis in search, of which :func:`returnn_amd.beam_search.beam_select` takes the best.

``python -m returnn_amd.language_model`` trains a small one on a made-up text on the GPU and completes it.
"""

from __future__ import annotations

import sys
from typing import List, NamedTuple, Optional, Tuple, Union

import torch

from .beam_search import beam_select, reorder_states
from .delta_rule import DeltaRecurrence
from .dropout import Dropout
from .embedding import Embedding
from .lstm import LSTM, LstmState
from .recurrence import GatedRecurrence
from .scoring import TokenScores, token_log_probs

__all__ = ["RecurrentLanguageModel", "Hypotheses"]


class Hypotheses(NamedTuple):
    """Of one search, the best first."""

    tokens: torch.Tensor  # [beam,length]
    log_probs: torch.Tensor  # [beam] of the tokens together, float32


class RecurrentLanguageModel(torch.nn.Module):
    """
    :param num_tokens: size of the vocabulary
    :param dim: width of the embedding and of every layer
    :param layer: "gated" (parallel in time), "delta" (likewise, with matrices as state) or "lstm"
    :param drop_prob: of the embedding and of every layer's output
    :param same_over_time: one dropout mask for all frames of a sequence
    """

    def __init__(
        self, num_tokens: int, dim: int, num_layers: int, *, layer: str = "gated", drop_prob: float = 0.0, same_over_time: bool = False, seed: int = 0,
        device=None, dtype=None,
    ):  # fmt: skip
        super().__init__()
        kinds = {"gated": GatedRecurrence, "delta": DeltaRecurrence, "lstm": LSTM}
        if layer not in kinds:
            raise ValueError("RecurrentLanguageModel: layer must be 'gated', 'delta' or 'lstm', got %r" % (layer,))
        self.num_tokens, self.dim = int(num_tokens), int(dim)
        kw = dict(device=device, dtype=dtype)
        self.embedding = Embedding(self.num_tokens, self.dim, **kw)
        self.layers = torch.nn.ModuleList(kinds[layer](self.dim, self.dim, **kw) for _ in range(int(num_layers)))
        # (a seed of its own for each, so that no two masks of a step are alike)
        self.dropouts = torch.nn.ModuleList(Dropout(drop_prob, seed=seed * 1009 + k, same_over_time=same_over_time) for k in range(int(num_layers) + 1))
        self.output = torch.nn.Linear(self.dim, self.num_tokens, **kw)

    def default_initial_state(self, *, batch_dims, device=None) -> list:
        """One state per layer: zeros."""
        return [m.default_initial_state(batch_dims=batch_dims, device=device) for m in self.layers]

    def logits(
        self, tokens: torch.Tensor, *, state: Optional[list] = None, seq_lens: Optional[torch.Tensor] = None, offset: Optional[Union[int, torch.Tensor]] = None
    ) -> Tuple[torch.Tensor, list]:
        """
        :param tokens: [T,B], or [B] for a single step
        :param offset: of the dropout masks (:class:`Dropout`; one for all of the model's, whose seeds differ), instead of each one's next.  On the GPU for a
            training step that is recorded into a graph.
        :return: logits of the next token [T,B,num_tokens] (or [B,num_tokens]), new state
        """
        if state is None:
            state = self.default_initial_state(batch_dims=(tokens.shape[-1],), device=tokens.device)
        x = self.dropouts[0](self.embedding(tokens), offset=offset)
        new_state = []
        for m, drop, s in zip(self.layers, self.dropouts[1:], state):
            y, s = m(x, state=s, seq_lens=seq_lens)
            new_state.append(s)
            x = drop(y, residual=x, offset=offset)
        return self.output(x), new_state

    def scores(
        self, tokens: torch.Tensor, targets: Optional[torch.Tensor] = None, *, state: Optional[list] = None, seq_lens: Optional[torch.Tensor] = None,
        entropy: bool = False, top_k: int = 0, offset: Optional[Union[int, torch.Tensor]] = None,
    ) -> Tuple[TokenScores, list]:  # fmt: skip
        """
        :param tokens: [T,B] or [B]
        :param targets: the tokens that followed, in the same shape; negative where there is none.  Frames past ``seq_lens`` have none.
        :return: :func:`token_log_probs` of the logits, new state
        """
        logits, state = self.logits(tokens, state=state, seq_lens=seq_lens, offset=offset)
        if targets is not None:
            targets = self._inside(targets, seq_lens)
        return token_log_probs(logits, targets, entropy=entropy, top_k=top_k), state

    @staticmethod
    def _inside(targets: torch.Tensor, seq_lens: Optional[torch.Tensor]) -> torch.Tensor:
        """The targets, [T,B] or [B], with none past the sequences' lengths."""
        if seq_lens is None:
            return targets
        frame = torch.arange(targets.shape[0], device=targets.device)[:, None] if targets.dim() == 2 else 0
        return torch.where(seq_lens.to(targets.device) > frame, targets, -1)

    def loss(
        self, tokens: torch.Tensor, targets: torch.Tensor, *, seq_lens: Optional[torch.Tensor] = None, entropy_scale: float = 0.0,
        offset: Optional[Union[int, torch.Tensor]] = None,
    ) -> torch.Tensor:  # fmt: skip
        """
        Cross entropy per token that there is, less ``entropy_scale`` times the entropy.

        :param tokens, targets: [T,B]; a negative target is none
        :param offset: as of :meth:`logits`
        """
        targets = self._inside(targets, seq_lens)
        logits, _ = self.logits(tokens, seq_lens=seq_lens, offset=offset)
        s = token_log_probs(logits, targets, entropy=entropy_scale != 0.0)
        total = -s.log_probs.sum()
        if entropy_scale:
            total = total - entropy_scale * s.entropy.sum()
        return total / (targets >= 0).sum().clamp(min=1)

    @torch.no_grad()
    def search(self, start: torch.Tensor, *, beam: int, length: int) -> Hypotheses:
        """
        The likeliest continuations, by beam search.

        :param start: [S] tokens, S >= 1
        :param beam: 1 to 64 hypotheses
        :param length: of the continuations
        """
        if start.dim() != 1 or start.numel() == 0:
            raise ValueError("search: start must be [S] tokens, S >= 1, got %s" % (tuple(start.shape),))
        if not 1 <= int(beam) <= 64:
            raise ValueError("search: beam must be 1 to 64, got %r" % (beam,))
        k = min(int(beam), self.num_tokens)  # alternatives of each hypothesis
        state = self.default_initial_state(batch_dims=(1,), device=start.device)
        if start.numel() > 1:
            _, state = self.logits(start[:-1, None], state=state)
        last, total = start[-1:], torch.zeros((1,), device=start.device)
        tokens = torch.empty((1, 0), dtype=torch.int64, device=start.device)
        for _ in range(int(length)):
            s, state = self.scores(last, state=state, top_k=k)
            total, source, at = beam_select(s.top_log_probs, total, min(int(beam), s.top_ids.numel()))
            last = s.top_ids[source, at]
            flat = [t for v in state for t in (v if isinstance(v, LstmState) else (v,))]
            tokens, *flat = reorder_states([tokens] + flat, source)
            tokens = torch.cat((tokens, last[:, None]), dim=1)
            flat = iter(flat)
            state = [LstmState(*(next(flat) for _ in v)) if isinstance(v, LstmState) else next(flat) for v in state]
        return Hypotheses(tokens, total)


def main(argv: Optional[List[str]] = None) -> int:
    """Train on a text that repeats itself, complete it."""
    import argparse

    ap = argparse.ArgumentParser(prog="python -m returnn_amd.language_model", description=main.__doc__)
    ap.add_argument("--layer", choices=["gated", "delta", "lstm"], default="gated")
    ap.add_argument("--steps", type=int, default=150)
    args = ap.parse_args(argv)
    if not torch.cuda.is_available():
        print("no GPU visible", file=sys.stderr)
        return 1
    torch.manual_seed(1)
    text = "the quick brown fox jumps over the lazy dog. "
    symbols = sorted(set(text))
    ids = torch.tensor([symbols.index(c) for c in text * 40], device="cuda")
    m = RecurrentLanguageModel(len(symbols), 128, 2, layer=args.layer, drop_prob=0.1, device="cuda")
    opt = torch.optim.Adam(m.parameters(), lr=3e-3)
    T, B = 64, 16
    for step in range(args.steps):
        first = torch.randint(0, ids.numel() - T - 1, (B,))
        tokens = torch.stack([ids[f : f + T + 1] for f in first.tolist()], dim=1)
        lens = torch.randint(T // 2, T + 1, (B,), device="cuda")
        opt.zero_grad()
        loss = m.loss(tokens[:-1], tokens[1:], seq_lens=lens)
        loss.backward()
        opt.step()
        if step % 50 == 0 or step == args.steps - 1:
            print("step %i: %.3f nats per token" % (step, float(loss.detach())), flush=True)
    m.eval()
    best = m.search(ids[:10], beam=4, length=35)
    print(text[:10] + "".join(symbols[t] for t in best.tokens[0].tolist()), "(%.2f)" % float(best.log_probs[0]))
    return 0


if __name__ == "__main__":
    sys.exit(main())
