"""The operators of whole language models as they are used together: the recurrent language model with matrices as state, in training, scoring and search."""

from __future__ import annotations

import math

import pytest
import torch

from _gpu_util import announce
from returnn_amd import language_model
from returnn_amd.beam_search import beam_select, reorder_states
from returnn_amd.delta_rule import gated_delta_rule
from returnn_amd.embedding import embed
from returnn_amd.language_model import RecurrentLanguageModel

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def model(V=23, dim=24, layers=2, **kw):
    torch.manual_seed(5)
    return RecurrentLanguageModel(V, dim, layers, layer="delta", device=DEV, **kw)


def test_loss_and_gradients_against_float64():
    """A stack of layers in float64 with autograd, on the CPU, frame by frame."""
    announce("model path gradients")
    T, B, V = 37, 4, 23
    m = model(V=V)
    tokens, targets, lens = torch.randint(0, V, (T, B)), torch.randint(0, V, (T, B)), torch.tensor([37, 4, 0, 33])
    loss = m.loss(tokens.to(DEV), targets.to(DEV), seq_lens=lens, entropy_scale=0.3)
    loss.backward()
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in m.named_parameters()}
    x = p["embedding.weight"][tokens]
    inside = (torch.arange(T)[:, None] < lens[None, :])[..., None]
    for n, layer in enumerate(m.layers):
        q, k, v, g, b = torch.nn.functional.linear(x, p["layers.%i.ff" % n], p["layers.%i.bias" % n]).split(layer.split, dim=-1)
        q, k = (t.unflatten(-1, (layer.num_heads, layer.key_dim)) for t in (q, k))
        q, k = (t * torch.rsqrt(t.square().sum(dim=-1, keepdim=True) + 1e-6) for t in (q, k))
        v, a, b = v.unflatten(-1, (layer.num_heads, layer.value_dim)), torch.exp(-torch.nn.functional.softplus(g)), torch.sigmoid(b)
        s, ys = torch.zeros((B, layer.num_heads, layer.key_dim, layer.value_dim), dtype=torch.float64), []
        for t in range(T):
            kept = a[t][..., None, None] * s
            missing = v[t] - (kept * k[t][..., None]).sum(-2)
            s = torch.where(inside[t][..., None, None], kept + k[t][..., None] * (b[t][..., None] * missing)[..., None, :], s)
            ys.append((s * q[t][..., None]).sum(-2).flatten(1) / math.sqrt(layer.key_dim))
        x = x + torch.where(inside, torch.stack(ys), 0.0)
    log_p = torch.log_softmax(torch.nn.functional.linear(x, p["output.weight"], p["output.bias"]), dim=-1)
    each = -log_p.gather(-1, targets[..., None])[..., 0] + 0.3 * (log_p.exp() * log_p).sum(-1)
    want = torch.where(inside[..., 0], each, 0.0).sum() / lens.sum()
    want.backward()
    # float32 against float64: sums of a few hundred terms, 1e-5 of the largest is hundreds of units in the last place
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * abs(float(want.detach()))
    for name, v in m.named_parameters():
        assert (v.grad.double().cpu() - p[name].grad).abs().max() <= 1e-5 * p[name].grad.abs().max().clamp(min=1e-3), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_are_the_sequence(dtype):
    """Scores of a text in one pass, and token by token with the state handed on."""
    announce("model path steps", dtype)
    T, B, V = 40, 3, 50
    m = model(V=V, dim=64, dtype=dtype).eval()
    tokens, targets = torch.randint(0, V, (T, B), device=DEV), torch.randint(0, V, (T, B), device=DEV)
    with torch.no_grad():
        whole, _ = m.scores(tokens, targets)
        state, each = None, []
        for t in range(T):
            s, state = m.scores(tokens[t], targets[t], state=state)
            each.append(s.log_probs)
    # (in bfloat16 every activation is rounded, on both sides: log probabilities of about 5 from logits good to 2^-6 of theirs)
    assert (whole.log_probs - torch.stack(each)).abs().max() <= (0.1 if dtype == torch.bfloat16 else 1e-4)


def test_search_against_all_continuations():
    """A beam that holds every hypothesis finds the best of all texts."""
    announce("model path search")
    V, length = 4, 3
    m = model(V=V, dim=16, layers=1).eval()
    start = torch.tensor([1, 2], device=DEV)
    best = m.search(start, beam=V ** (length - 1), length=length)
    texts = torch.cartesian_prod(*[torch.arange(V)] * length).to(DEV)
    line = torch.cat((start[:, None].expand(-1, len(texts)), texts.t()))
    with torch.no_grad():
        s, _ = m.scores(line[:-1], line[1:])
    total = s.log_probs[start.numel() - 1 :].sum(0)
    order = total.argsort(descending=True)[: len(best.tokens)]
    assert torch.equal(best.tokens[0], texts[order[0]]) and (best.log_probs - total[order]).abs().max() < 1e-4


@pytest.mark.parametrize("layer", ["gated", "lstm", "delta"])
def test_a_batch_of_searches(layer):
    """Searches side by side, with an end: selection and reordering on the axis of the searches, against each by itself."""
    announce("model path batch of searches", layer)
    torch.manual_seed(8)
    V, K, B, end, length = 30, 4, 3, 7, 6
    m = RecurrentLanguageModel(V, 32, 2, layer=layer, device=DEV).eval()

    def states(flat, shape):
        return [t.reshape(shape + tuple(t.shape[t.dim() - (t.dim() - 1) :])) for t in flat]

    def run(first):
        n = first.numel()
        state = m.default_initial_state(batch_dims=(n * K,), device=DEV)
        kind = type(state[0])
        totals = torch.full((n, K), -math.inf, device=DEV)
        totals[:, 0] = 0.0
        last, ended = first[:, None].expand(n, K), torch.zeros((n, K), dtype=torch.bool, device=DEV)
        texts = torch.zeros((n, K, 0), dtype=torch.int64, device=DEV)
        for _ in range(length):
            logits, state = m.logits(last.reshape(-1), state=state)
            step = beam_select(torch.log_softmax(logits.float(), -1).view(n, K, V), totals, K, ended=ended, end_token=end)
            flat = [t for v in state for t in (v if isinstance(v, tuple) else (v,))]
            ended, texts, *flat = reorder_states([ended, texts] + states(flat, (n, K)), step.sources)
            flat = [t.flatten(0, 1) for t in flat]
            state = [kind(*flat[2 * i : 2 * i + 2]) for i in range(len(m.layers))] if issubclass(kind, tuple) else flat
            totals, last = step.totals, step.tokens
            ended, texts = ended | (last == end), torch.cat((texts, last[..., None]), dim=-1)
        return totals, texts

    with torch.no_grad():
        first = torch.tensor([2, 9, 21], device=DEV)
        totals, texts = run(first)
        assert (totals[:, :-1] >= totals[:, 1:]).all() and torch.isfinite(totals).all()
        after = (texts == end).cumsum(-1) - (texts == end).int() > 0
        assert (texts[after] == end).all()
        for n in range(B):
            t, x = run(first[n : n + 1])
            # (the projection's products may be added in another order for another number of rows)
            assert (t[0] - totals[n]).abs().max() < 1e-4 and torch.equal(x[0, 0], texts[n, 0])


def test_in_a_region_and_recorded():
    """A training step in an autocast region; one that is recorded into a graph, replayed on other tokens."""
    announce("model path region and graph")
    T, B, V = 33, 4, 40
    m = model(V=V, dim=64, drop_prob=0.2)
    gen = torch.Generator(device=DEV).manual_seed(3)
    tokens, targets = torch.randint(0, V, (T, B), device=DEV, generator=gen), torch.randint(0, V, (T, B), device=DEV, generator=gen)
    lens = torch.tensor([33, 5, 20, 1], device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = m.loss(tokens, targets, seq_lens=lens)
    loss.backward()
    for name, p in m.named_parameters():
        assert p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() and p.grad.any(), name
    del loss
    offset = torch.zeros((), dtype=torch.int64, device=DEV)
    leaves = list(m.parameters())

    def step():
        return torch.autograd.grad(m.loss(tokens, targets, seq_lens=lens, offset=offset), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for n in range(3):
        offset.fill_(n + 1)
        tokens.copy_(torch.randint(0, V, (T, B), device=DEV, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        # (torch's own matrix products may choose another way outside the graph)
        for a, b in zip(step(), recorded):
            assert (a - b).abs().max() <= 1e-5 * a.abs().max()


def test_the_program_runs(capsys):
    announce("model path program")
    assert language_model.main(["--layer", "delta", "--steps", "3"]) == 0
    assert "nats per token" in capsys.readouterr().out


def test_views_that_are_to_be_negated():
    """The imaginary part of a conjugated tensor is a view whose numbers lie in memory with the other sign."""
    announce("model path negated views")
    gen = torch.Generator(device=DEV).manual_seed(7)

    def negated(*shape):
        v = torch.view_as_complex(torch.randn(shape + (2,), device=DEV, generator=gen)).conj().imag
        assert v.is_neg()
        return v, v.resolve_neg().contiguous()

    for T in (5, 40):
        (q, q1), (v, v1) = negated(T, 2, 1, 8), negated(T, 2, 1, 8)
        k = torch.nn.functional.normalize(torch.randn((T, 2, 1, 8), device=DEV, generator=gen), dim=-1)
        g, b = -torch.rand((T, 2, 1), device=DEV, generator=gen), torch.rand((T, 2, 1), device=DEV, generator=gen)
        assert all(torch.equal(x, y) for x, y in zip(gated_delta_rule(q, k, v, g, b), gated_delta_rule(q1, k, v1, g, b)))
    (w, w1), tokens = negated(9, 6), torch.tensor([2, 8, -1], device=DEV)
    assert torch.equal(embed(tokens, w), embed(tokens, w1))
    (scores, scores1), (totals, totals1) = negated(2, 3, 50), negated(2, 3)
    a, b = beam_select(scores, totals, 4), beam_select(scores1, totals1, 4)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    state = torch.view_as_complex(torch.randn((2, 3, 5, 2), device=DEV, generator=gen)).conj()
    for s in (state, state.imag, scores):
        (r,) = reorder_states([s], a.sources)
        assert torch.equal(r, s[torch.arange(2, device=DEV)[:, None], a.sources])


def test_calls_side_by_side():
    """Two streams with the same calls on other numbers, each with workspaces of its own."""
    announce("model path two streams")
    gen = torch.Generator(device=DEV).manual_seed(9)
    jobs = []
    for _ in range(2):
        q, k, v = (torch.nn.functional.normalize(torch.randn((700, 2, 2, 32), device=DEV, generator=gen), dim=-1) for _ in "qkv")
        g, b = -torch.rand((700, 2, 2), device=DEV, generator=gen), torch.rand((700, 2, 2), device=DEV, generator=gen)
        jobs.append((q, k, v, g, b, torch.randint(0, 900, (10000,), device=DEV, generator=gen), torch.randn((900, 33), device=DEV, generator=gen),
                     torch.randn((10000, 33), device=DEV, generator=gen), torch.randn((3, 40, 9000), device=DEV, generator=gen), torch.randn((3, 40), device=DEV, generator=gen)))  # fmt: skip

    def run(q, k, v, g, b, tokens, w, dy, scores, totals):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, g, b, w)]
        y, s = gated_delta_rule(*leaves[:5])
        x = embed(tokens, leaves[5])
        step = beam_select(scores, totals, 64)
        return (y, s, x) + torch.autograd.grad((y, s, x), leaves, (v, s.detach(), dy)) + tuple(step) + tuple(reorder_states([totals], step.sources))

    want = [run(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for stream, j in zip(streams, jobs):
            with torch.cuda.stream(stream):
                got.append(run(*j))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, r in zip(want, got) for a, b in zip(w, r))
