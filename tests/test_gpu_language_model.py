"""The recurrent language model: the sequence operators together, in training, scoring and search."""

from __future__ import annotations

import itertools

import numpy
import pytest
import torch

from _gpu_util import announce
from returnn_amd import language_model
from returnn_amd.language_model import RecurrentLanguageModel

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def model(layer="gated", V=23, dim=12, layers=2, **kw):
    torch.manual_seed(5)
    return RecurrentLanguageModel(V, dim, layers, layer=layer, device=DEV, **kw)


def test_loss_and_gradients_against_float64():
    """A stack of gated layers in float64 with autograd, on the CPU."""
    announce("language model gradients")
    T, B, V = 9, 4, 23
    m = model(V=V)
    tokens, targets, lens = torch.randint(0, V, (T, B)), torch.randint(0, V, (T, B)), torch.tensor([9, 4, 0, 7])
    loss = m.loss(tokens.to(DEV), targets.to(DEV), seq_lens=lens, entropy_scale=0.3)
    loss.backward()
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in m.named_parameters()}
    x = p["embedding.weight"][tokens]
    inside = (torch.arange(T)[:, None] < lens[None, :])[..., None]
    for k in range(2):
        gates = torch.nn.functional.linear(x, p["layers.%i.ff" % k], p["layers.%i.bias" % k])
        c, ys = torch.zeros((B, m.dim), dtype=torch.float64), []
        for t in range(T):
            z, i, f, o = gates[t].chunk(4, dim=-1)
            c = torch.where(inside[t], torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(z), c)
            ys.append(torch.where(inside[t], torch.sigmoid(o) * c, 0.0))
        x = x + torch.stack(ys)
    log_p = torch.log_softmax(torch.nn.functional.linear(x, p["output.weight"], p["output.bias"]), dim=-1)
    each = -log_p.gather(-1, targets[..., None])[..., 0] + 0.3 * (log_p.exp() * log_p).sum(-1)
    want = torch.where(inside[..., 0], each, 0.0).sum() / lens.sum()
    want.backward()
    # float32 against float64: sums of a few hundred terms, 1e-5 of the largest is hundreds of units in the last place
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * abs(float(want.detach()))
    for name, v in m.named_parameters():
        assert (v.grad.double().cpu() - p[name].grad).abs().max() <= 1e-5 * p[name].grad.abs().max().clamp(min=1e-3), name


@pytest.mark.parametrize("layer", ["gated", "lstm"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_are_the_sequence(layer, dtype):
    """Scores of a text in one pass, and token by token with the state handed on."""
    announce("language model steps", layer, dtype)
    T, B, V = 17, 3, 50
    m = model(layer, V=V, dim=32, dtype=dtype).eval()
    tokens, targets = torch.randint(0, V, (T, B), device=DEV), torch.randint(0, V, (T, B), device=DEV)
    with torch.no_grad():
        whole, _ = m.scores(tokens, targets, entropy=True, top_k=5)
        state = None
        for t in range(T):
            one, state = m.scores(tokens[t], targets[t], state=state, entropy=True, top_k=5)
            # (bfloat16: layers, sums and logits each rounded to 2^-8, in products of another order)
            bound = 1e-4 if dtype == torch.float32 else 0.1
            assert (one.log_probs - whole.log_probs[t]).abs().max() < bound and (one.entropy - whole.entropy[t]).abs().max() < bound


def test_frames_without_a_target():
    """They are not among the tokens that the loss is a mean over; and a step of sequences that have ended has none."""
    announce("language model frames without a target")
    T, B, V = 6, 3, 30
    m = model(V=V).eval()
    tokens, targets, lens = torch.randint(0, V, (T, B), device=DEV), torch.randint(0, V, (T, B), device=DEV), torch.tensor([6, 3, 5])
    targets[1, 0] = targets[0, 1] = -1
    with torch.no_grad():
        whole, _ = m.scores(tokens, targets, seq_lens=lens)
        # (two orders of 12 float32 terms)
        assert abs(float(m.loss(tokens, targets, seq_lens=lens)) + float(whole.log_probs.sum()) / 12) < 1e-5
        one, _ = m.scores(tokens[0], targets[0], seq_lens=torch.tensor([1, 1, 0]))
        assert float(one.log_probs[0]) < 0 and one.log_probs[1:].tolist() == [0.0, 0.0]
        assert float(m.loss(tokens, torch.full_like(targets, -1))) == 0.0


def test_dropout_repeats_with_its_offsets():
    announce("language model dropout")
    m = model(V=40, dim=24, drop_prob=0.3)
    tokens, targets = torch.randint(0, 40, (12, 5), device=DEV), torch.randint(0, 40, (12, 5), device=DEV)

    def step():
        m.zero_grad()
        loss = m.loss(tokens, targets)
        loss.backward()
        return [loss.detach().clone()] + [p.grad.clone() for p in m.layers.parameters()]

    first, second = step(), step()
    assert not torch.equal(first[0], second[0])
    for d in m.dropouts:
        d.offset = 0
    for a, b in zip(step(), first):
        assert torch.equal(a, b)
    m.eval()
    assert torch.equal(m.loss(tokens, targets), m.loss(tokens, targets))


@pytest.mark.parametrize("layer", ["gated", "lstm"])
def test_search_finds_the_best_of_all(layer):
    """A beam as wide as all continuations but the last token: the best one of all is in it."""
    announce("language model search", layer)
    V, length = 4, 3
    m = model(layer, V=V, dim=16).eval()
    start = torch.tensor([1, 3], device=DEV)
    got = m.search(start, beam=V ** (length - 1), length=length)
    texts = torch.tensor(list(itertools.product(range(V), repeat=length)), device=DEV).t()
    full = torch.cat((start[:, None].expand(2, texts.shape[1]), texts))
    with torch.no_grad():
        s, _ = m.scores(full[:-1], full[1:])
    total = s.log_probs[1:].sum(0)
    assert torch.equal(got.tokens[0], texts[:, int(total.argmax())])
    assert abs(float(got.log_probs[0]) - float(total.max())) < 1e-4
    assert got.tokens.shape == (V ** (length - 1), length)
    for bad in (dict(start=start[:0], beam=2), dict(start=start, beam=0), dict(start=start, beam=65)):
        with pytest.raises(ValueError):
            m.search(**bad, length=1)
    with pytest.raises(ValueError):
        RecurrentLanguageModel(5, 4, 1, layer="gru")


def test_the_example_learns(capsys):
    announce("language model example")
    assert language_model.main(["--steps", "120"]) == 0
    lines = [line for line in capsys.readouterr().out.splitlines() if not line.startswith("[gpu case]")]
    first, last = (float(line.split(": ")[1].split()[0]) for line in (lines[0], lines[-2]))
    assert numpy.isfinite(last) and last < 0.5 * first
