"""The sequence operators in torch's modes that are not plain calls: forward derivatives, autocast regions, recomputed segments, recorded steps."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.utils.checkpoint import checkpoint

from _gpu_util import announce
from returnn_amd.dropout import Dropout, dropout
from returnn_amd.language_model import RecurrentLanguageModel
from returnn_amd.recurrence import GatedRecurrence, gated_recurrence
from returnn_amd.scoring import token_log_probs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("grad_mode", [True, False])
def test_a_tangent_is_not_lost(grad_mode):
    """No operator has a derivative in forward mode: inputs that have a tangent are refused, as torch's own functions without one do."""
    announce("sequence modes tangent", grad_mode)
    x = torch.randn((5, 3, 8), device=DEV)
    c0, r = torch.randn((3, 2), device=DEV), torch.randn_like(x)
    targets = torch.zeros((5, 3), dtype=torch.int64, device=DEV)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        dual = {k: forward_ad.make_dual(t, torch.ones_like(t)) for k, t in (("x", x), ("c0", c0), ("r", r))}
        for call in (
            lambda: gated_recurrence(dual["x"]), lambda: gated_recurrence(dual["x"][0]), lambda: gated_recurrence(x, state=dual["c0"]),
            lambda: dropout(dual["x"], 0.5, seed=1), lambda: dropout(x, 0.5, seed=1, residual=dual["r"]),
            lambda: token_log_probs(dual["x"], targets), lambda: token_log_probs(dual["x"], top_k=2),
        ):  # fmt: skip
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        gated_recurrence(x, state=c0)  # (what has no tangent is taken in a dual level as well)
        dropout(x, 0.5, seed=1, residual=r)
        token_log_probs(x, targets)


def _layer_output(amp, gates):
    """The type in which the operators take a projection of the region."""
    return gates if amp == torch.bfloat16 else gates.float()


@pytest.mark.parametrize("amp", [torch.bfloat16, torch.float16], ids=str)
def test_results_of_products_of_a_region(amp):
    """Float16 is taken as float32 inside a region (and refused outside, see the operators' refusals); values and gradients are those of the cast."""
    announce("sequence modes autocast operators", amp)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((7, 3, 16), device=DEV, generator=gen).to(amp).requires_grad_()
    r = torch.randn((7, 3, 16), device=DEV, generator=gen).to(amp).requires_grad_()
    targets = torch.randint(0, 16, (7, 3), device=DEV, generator=gen)
    calls = (
        lambda x, r: gated_recurrence(x, seq_lens=torch.tensor([7, 2, 5]), direction=-1), lambda x, r: gated_recurrence(x[0]),
        lambda x, r: (dropout(x, 0.4, seed=5, residual=r),), lambda x, r: token_log_probs(x, targets, entropy=True, top_k=3)[:2],
    )  # fmt: skip
    for call in calls:
        with torch.autocast("cuda", dtype=amp):
            got = call(x, r)
        want = call(_layer_output(amp, x), _layer_output(amp, r))
        for a, b in zip(got, want):
            assert a.dtype == b.dtype and torch.equal(a, b)
        errors = [torch.randn_like(a) for a in got]
        for a, b in zip(torch.autograd.grad(got, (x, r), errors, allow_unused=True), torch.autograd.grad(want, (x, r), errors, allow_unused=True)):
            assert (a is None) == (b is None) and (a is None or (a.dtype == amp and torch.equal(a, b)))


@pytest.mark.parametrize("layer", ["gated", "lstm"])
@pytest.mark.parametrize("amp", [torch.bfloat16, torch.float16], ids=str)
def test_language_model_in_a_region(amp, layer):
    """A training step and search of a float32 model: the layers' outputs are added to a float32 stream, as they are in evaluation."""
    announce("sequence modes autocast model", amp, layer)
    torch.manual_seed(6)
    T, B, V, dim = 9, 4, 30, 32
    m = RecurrentLanguageModel(V, dim, 2, layer=layer, drop_prob=0.3, seed=4, device=DEV)
    tokens, targets, lens = torch.randint(0, V, (T, B), device=DEV), torch.randint(0, V, (T, B), device=DEV), torch.tensor([9, 4, 1, 7])
    with torch.autocast("cuda", dtype=amp):
        loss = m.loss(tokens, targets, seq_lens=lens, entropy_scale=0.1)
    loss.backward()
    assert loss.dtype == torch.float32 and torch.isfinite(loss)
    for name, p in m.named_parameters():
        assert p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() and p.grad.any(), name
    # the same, operator by operator
    with torch.autocast("cuda", dtype=amp), torch.no_grad():
        x = dropout(m.embedding(tokens), 0.3, seed=m.dropouts[0].seed)
        for k, sub in enumerate(m.layers):
            y, _ = sub(x, state=sub.default_initial_state(batch_dims=(B,)), seq_lens=lens)
            assert y.dtype == (torch.bfloat16 if amp == torch.bfloat16 else torch.float32)
            x = dropout(y.float(), 0.3, seed=m.dropouts[k + 1].seed, residual=x)
        logits = m.output(x)
        assert logits.dtype == amp
        inside = torch.arange(T, device=DEV)[:, None] < lens.to(DEV)
        s = token_log_probs(_layer_output(amp, logits), torch.where(inside, targets, -1), entropy=True)
        assert torch.equal(loss.detach(), (-s.log_probs.sum() - 0.1 * s.entropy.sum()) / inside.sum())
        m.eval()
        whole, _ = m.scores(tokens, targets)
        assert whole.log_probs.dtype == torch.float32 and m.search(tokens[:3, 0], beam=5, length=4).tokens.shape == (5, 4)


def test_types_that_differ_are_added_as_in_evaluation():
    announce("sequence modes residual types")
    m = Dropout(0.5, seed=2)
    x, r = torch.randn((4, 33), device=DEV), torch.randn((4, 33), device=DEV)
    for a, b in ((x.bfloat16(), r), (x, r.bfloat16())):
        m.offset = 0
        y = m.train()(a, residual=b)
        assert y.dtype == torch.float32 == m.eval()(a, residual=b).dtype
        assert torch.equal(y, dropout(a.float(), 0.5, seed=2, residual=b.float()))


def test_a_recorded_step_draws_anew():
    """A training step of the language model in a graph: every replay takes the offset that lies on the GPU, and gives what an eager step with it gives."""
    announce("sequence modes recorded step")
    torch.manual_seed(8)
    T, B, V = 12, 3, 40
    m = RecurrentLanguageModel(V, 64, 2, drop_prob=0.3, device=DEV)
    tokens, targets = torch.randint(0, V, (T, B), device=DEV), torch.randint(0, V, (T, B), device=DEV)
    lens = torch.tensor([12, 5, 9], device=DEV)
    offset = torch.zeros((1,), dtype=torch.int64, device=DEV)
    weights = [p for k, p in m.named_parameters() if k.startswith("layers")]

    def step(offset):
        loss = m.loss(tokens, targets, seq_lens=lens, offset=offset)
        return (loss.detach(),) + torch.autograd.grad(loss, weights)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(offset)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(offset)
    seen = []
    for k in (3, 0, 1 << 40, 4):
        want = step(k)
        torch.cuda.synchronize()
        offset.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k
        seen.append(float(out[0]))
    assert len(set(seen)) == 4 and all(d.offset == 0 for d in m.dropouts)


def test_the_modules_own_offset_is_not_recorded():
    announce("sequence modes recorded module")
    m, x = Dropout(0.5, seed=3), torch.ones((4, 64), device=DEV)
    offset = torch.full((1,), 7, dtype=torch.int64, device=DEV)
    want = dropout(x, 0.5, seed=3, offset=7)
    assert torch.equal(m(x, offset=7), want) and torch.equal(m(x, offset=offset), want) and m.offset == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="replay"):
            m(x)
        y = m(x, residual=x, offset=offset)
        z = m.eval()(x, residual=x)
    graph.replay()
    torch.cuda.synchronize()
    assert m.offset == 0 and torch.equal(y, want + x) and torch.equal(z, x + x)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_segments(reentrant):
    """With an offset of its own a segment's gradients are those without recomputation; the module's next one would be another mask and is refused."""
    announce("sequence modes recomputed", reentrant)
    torch.manual_seed(9)
    m, layer = Dropout(0.5, seed=3), GatedRecurrence(24, 24, device=DEV)
    x, dy = torch.randn((9, 4, 24), device=DEV, requires_grad=True), torch.randn((9, 4, 24), device=DEV)

    def segment(x, offset):
        y, _ = layer(m(x, offset=offset))
        return m(y, residual=x, offset=offset + 1000)

    def gradients(y):
        for t in (x, *layer.parameters()):
            t.grad = None
        y.backward(dy)
        return tuple(t.grad.clone() for t in (x, *layer.parameters()))

    want = segment(x, 5)
    plain = gradients(want)
    y = checkpoint(segment, x, 5, use_reentrant=reentrant)
    assert torch.equal(y, want)
    for a, b in zip(gradients(y), plain):
        assert torch.equal(a, b)
    y = checkpoint(lambda x: layer(m(x))[0], x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="recomputed"):
        gradients(y)
    assert m.offset == 1
    torch.autograd.grad(m(x), x, dy)  # (nothing of the refusal is left)
    assert m.offset == 2
