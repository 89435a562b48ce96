"""Embedding with scaling and its gradient against their definition in float64, on cuda:0."""

from __future__ import annotations

import numpy
import pytest
import torch

import _model_ref as ref
from _gpu_util import announce
from returnn_amd.embedding import Embedding, embed

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(tokens, V, D, dtype, *, scale=1.0, seed=1):
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn((V, D), generator=gen).to(dtype).to(DEV).requires_grad_()
    dy = torch.randn(tuple(tokens.shape) + (D,), generator=gen).to(dtype).to(DEV)
    tokens = tokens.to(DEV)
    y = embed(tokens, w, scale=scale)
    (d,) = torch.autograd.grad(y, w, dy)
    assert y.dtype == d.dtype == dtype and y.shape == dy.shape and d.shape == w.shape
    half = torch.finfo(dtype).eps / 2  # one rounding of the result
    a = w.detach().double().cpu().numpy()
    want = ref.embed(tokens.cpu().numpy(), a, scale)
    got = y.detach().double().cpu().numpy()
    assert numpy.array_equal(numpy.isnan(got), numpy.isnan(want))
    # (the product is rounded to float32 first)
    assert (abs(got - want)[~numpy.isnan(want)] <= ((half + 2.0**-24) * abs(want) + 1e-40)[~numpy.isnan(want)]).all()
    want, most, count = ref.embed_grad(tokens.cpu().numpy(), dy.double().cpu().numpy(), V, scale)
    got = d.double().cpu().numpy()
    assert not got[count == 0].any()
    # (a sum of n numbers in float32 is off by (n - 1) 2^-24 of the sum of their absolute values at most, and scaled and rounded once)
    assert (abs(got - want) <= half * abs(want) + (count[:, None] + 2) * 2.0**-24 * most * (1 + half) + 1e-40).all()
    return y, d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("D", [1, 3, 7, 8, 9, 16, 31, 64, 100, 501, 512, 520, 1024, 1500])
def test_widths(D, dtype):
    announce("embedding widths", D, dtype)
    gen = torch.Generator().manual_seed(D)
    check(torch.randint(-1, 31, (57,), generator=gen), 29, D, dtype, scale=D**0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows", [0, 1, 7, 8, 9, 16, 17, 255, 256, 257, 4096, 8191, 8192, 8193, 12288, 20000])
def test_rows(rows, dtype):
    """Counted up to 8192 rows, sorted by digits beyond; tokens of different frequency, one of them a tenth of all."""
    announce("embedding rows", rows, dtype)
    gen = torch.Generator().manual_seed(rows)
    tokens = torch.randint(0, 700, (rows,), generator=gen)
    tokens = torch.where(torch.rand((rows,), generator=gen) < 0.1, 333, tokens)
    check(torch.where(torch.rand((rows,), generator=gen) < 0.2, -1, tokens), 700, 24, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,D", [(70000, 24), (33000, 600), (20000, 600), (66000, 3)])
def test_many_rows(rows, D, dtype):
    """Pieces of 16 and 32 rows."""
    announce("embedding many rows", rows, D, dtype)
    gen = torch.Generator().manual_seed(rows)
    tokens = torch.randint(-1, 900, (rows,), generator=gen)
    check(torch.where(torch.rand((rows,), generator=gen) < 0.05, 333, tokens), 890, D, dtype)


@pytest.mark.parametrize("V", [1, 2, 255, 256, 511, 512, 513, 70000, 262143, 262144])
@pytest.mark.parametrize("rows", [300, 9000])
def test_vocabularies(V, rows):
    announce("embedding vocabularies", V, rows)
    gen = torch.Generator().manual_seed(V)
    tokens = torch.randint(0, V, (rows,), generator=gen)
    tokens[:3] = torch.tensor([V - 1, 0, V])
    check(tokens, V, 12, torch.float32, scale=0.5)


@pytest.mark.parametrize("rows", [1000, 8192, 30000])
@pytest.mark.parametrize("D", [8, 40, 700])
def test_one_token_only(rows, D):
    """All rows of one token: a run over all pieces, and its errors added in order; whole numbers are added exactly."""
    announce("embedding one token", rows, D)
    check(torch.full((rows,), 2), 5, D, torch.bfloat16)
    tokens = torch.full((rows,), 3, device=DEV)
    tokens[rows // 2] = 1
    w = torch.zeros((5, D), device=DEV, requires_grad=True)
    dy = (torch.arange(rows, device=DEV) % 7).float()[:, None].expand(rows, D).contiguous()
    (d,) = torch.autograd.grad(embed(tokens, w), w, dy)
    total = (torch.arange(rows) % 7).sum() - rows // 2 % 7
    assert (d[3] == total).all() and (d[1] == rows // 2 % 7).all() and not d[[0, 2, 4]].any()


def test_order_does_not_change():
    """Repeated calls agree bit for bit, and so does one with the table's other rows in use or not."""
    announce("embedding repeated")
    gen = torch.Generator(device=DEV).manual_seed(4)
    for rows in (3000, 20000):
        tokens = torch.randint(0, 50, (rows,), device=DEV, generator=gen)
        w = torch.zeros((60, 200), device=DEV, requires_grad=True)
        dy = torch.randn((rows, 200), device=DEV, generator=gen)
        runs = [torch.autograd.grad(embed(tokens, w), w, dy)[0] for _ in range(4)]
        assert all(torch.equal(runs[0], r) for r in runs[1:])


@pytest.mark.parametrize("rows,D", [(3000, 200), (3000, 8), (3000, 40), (8192, 512), (20000, 200), (20000, 1500), (70000, 16)])
def test_other_tokens_do_not_change_a_sum(rows, D):
    """The rows of one token stay, those of others become other tokens: the token's sum is the same bit for bit."""
    announce("embedding other tokens", rows, D)
    gen = torch.Generator(device=DEV).manual_seed(rows + D)
    tokens = torch.randint(0, 50, (rows,), device=DEV, generator=gen)
    tokens[torch.rand((rows,), device=DEV, generator=gen) < 0.2] = 20
    dy = torch.randn((rows, D), device=DEV, generator=gen)
    w = torch.zeros((60, D), device=DEV, requires_grad=True)
    keep = (tokens == 20) | (tokens == 31)
    want = torch.autograd.grad(embed(tokens, w), w, dy)[0]
    for low, high in ((0, 20), (40, 60), (32, 60), (0, 5)):
        others = torch.randint(low, high, (rows,), device=DEV, generator=gen)
        got = torch.autograd.grad(embed(torch.where(keep, tokens, others), w), w, dy)[0]
        assert torch.equal(got[20], want[20]) and torch.equal(got[31], want[31])


def test_padding_is_not_read():
    announce("embedding padding")
    tokens = torch.tensor([[0, -1, 2], [-7, 1, 5]], device=DEV)
    w = torch.randn((3, 10), device=DEV, requires_grad=True)
    dy = torch.randn((2, 3, 10), device=DEV)
    dy[0, 1], dy[1, 0], dy[1, 2] = float("nan"), float("inf"), float("nan")
    y = embed(tokens, w)
    assert torch.isnan(y[1, 2]).all() and not y[0, 1].any() and not y[1, 0].any()
    (d,) = torch.autograd.grad(y, w, dy)
    assert torch.equal(d, torch.stack((dy[0, 0], dy[1, 1], dy[0, 2])))
    w = torch.randn((0, 10), device=DEV, requires_grad=True)
    y = embed(tokens, w)
    assert torch.isnan(y[tokens >= 0]).all() and not y[tokens < 0].any()
    assert torch.autograd.grad(y, w, dy)[0].shape == (0, 10)


def test_tables_and_errors_with_a_pitch():
    announce("embedding pitch")
    gen = torch.Generator(device=DEV).manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn((40, 37), device=DEV, generator=gen).to(dtype).requires_grad_()
        tokens = torch.randint(0, 40, (6, 50), device=DEV, generator=gen)
        dy = torch.randn((6, 50, 40), device=DEV, generator=gen).to(dtype)[..., 3:34]
        y = embed(tokens, wide[:, 2:33], scale=3.0)
        (d,) = torch.autograd.grad(y, wide, dy)
        leaf = wide.detach()[:, 2:33].clone().requires_grad_()
        z = embed(tokens.to(torch.int32), leaf, scale=3.0)
        assert torch.equal(y, z)
        assert torch.equal(d[:, 2:33], torch.autograd.grad(z, leaf, dy.contiguous())[0]) and not d[:, :2].any() and not d[:, 33:].any()
        y, z = (embed(t, leaf) for t in (tokens.t(), tokens.t().contiguous()))
        assert torch.equal(y, z)
        # an error that is one number for all, and one of transposed frames
        for e in (torch.ones((), dtype=dtype, device=DEV).expand(50, 6, 31), dy.transpose(0, 1)):
            assert torch.equal(torch.autograd.grad(y, leaf, e, retain_graph=True)[0], torch.autograd.grad(z, leaf, e.contiguous(), retain_graph=True)[0])


def test_offsets_beyond_32_bits():
    """A table of more than 2^32 elements: its last rows, forward and in the gradient."""
    announce("embedding large table")
    V, D = 300_000, 16384
    w = torch.zeros((V, D), dtype=torch.bfloat16, device=DEV)
    w[-1], w[-2] = 2.0, 3.0
    tokens = torch.tensor([V - 1, 5, V - 2, V - 1], device=DEV)
    y = embed(tokens, w.requires_grad_())
    assert y[:, 7].tolist() == [2.0, 0.0, 3.0, 2.0]
    (d,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert d[-1].eq(2).all() and d[-2].eq(1).all() and d[5].eq(1).all() and int(torch.count_nonzero(d[:, 0])) == 3 and not d[100_000].any() and not d[V - 3].any()


def test_another_stream_and_recorded_steps():
    announce("embedding streams and graphs")
    gen = torch.Generator(device=DEV).manual_seed(6)
    for rows in (500, 10000):
        w = torch.randn((300, 70), device=DEV, generator=gen, requires_grad=True)
        tokens, dy = torch.randint(-1, 300, (rows,), device=DEV, generator=gen), torch.randn((rows, 70), device=DEV, generator=gen)

        def step(w):
            y = embed(tokens, w, scale=2.0)
            return (y,) + torch.autograd.grad(y, w, dy)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(w)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            recorded = step(w)
        for _ in range(3):
            tokens.copy_(torch.randint(-1, 300, (rows,), device=DEV, generator=gen))
            graph.replay()
            torch.cuda.synchronize()
            want = step(w.detach().clone().requires_grad_())
            assert all(torch.equal(a, b) for a, b in zip(want, recorded))


def test_module_and_refusals():
    announce("embedding module")
    m = Embedding(11, 6, scale=0.5, device=DEV)
    tokens = torch.tensor([3, 3, -1, 10], device=DEV)
    assert torch.equal(m(tokens), torch.where((tokens >= 0)[:, None], 0.5 * m.weight.detach()[tokens.clamp(min=0)], 0.0))
    m(tokens).sum().backward()
    assert m.weight.grad[3].eq(1.0).all() and m.weight.grad[10].eq(0.5).all()
    w = m.weight.detach()
    for match, args in (
        ("tokens of type", (tokens.float(), w)), ("tokens of type", (tokens > 0, w)), ("table must be", (tokens, w[0])), ("float32 or bfloat16", (tokens, w.half())), ("is on", (tokens.cpu(), w)),
    ):  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            embed(*args)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(m(tokens).sum(), m.weight, create_graph=True)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        embed(tokens, torch.autograd.forward_ad.make_dual(w, w))
    assert embed(tokens[0], w).shape == (6,) and embed(tokens[:0], w).shape == (0, 6)
    leaf = w.clone().requires_grad_()
    embed(tokens[0], leaf, scale=2.0).sum().backward()  # (one token by itself)
    assert leaf.grad[3].eq(2.0).all() and int(leaf.grad.count_nonzero()) == 6
