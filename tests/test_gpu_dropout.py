"""
Dropout from a counter on the GPU against its definition: the mask is a whole-number matter and has to be the definition's
everywhere, the values have one product, one sum and one rounding (u = 2^-24; 2^-8 in bfloat16) each.
"""

from __future__ import annotations

import numpy
import pytest
import torch

import _sequence_ref as ref
from _gpu_util import announce
from returnn_amd.dropout import Dropout, dropout

pytestmark = pytest.mark.gpu
U = 2.0**-24
DEV = "cuda:0"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def array(t):
    return t.detach().double().cpu().numpy()


def check(y, x, factors, residual=None):
    want = array(x) * factors + (0.0 if residual is None else array(residual))
    size = numpy.abs(array(x) * factors) + (0.0 if residual is None else numpy.abs(array(residual)))
    half = 2.0**-8 if y.dtype == torch.bfloat16 else U
    assert numpy.all(numpy.abs(array(y) - want) <= 4 * U * size + half * numpy.abs(want))
    if residual is None:
        assert numpy.array_equal(array(y) != 0, (factors != 0) & (array(x) != 0))


def run(shape, dtype, p, *, seed=0x123456789ABCDEF, offset=5, residual=False, same=False):
    gen = torch.Generator(device=DEV).manual_seed(hash((shape, p)) & 0xFFFF)
    x = torch.randn(shape, device=DEV, generator=gen).to(_DTYPES[dtype]).requires_grad_()
    r = torch.randn(shape, device=DEV, generator=gen).to(_DTYPES[dtype]).requires_grad_() if residual else None
    dy = torch.randn(shape, device=DEV, generator=gen).to(_DTYPES[dtype])
    y = dropout(x, p, seed=seed, offset=offset, residual=r, same_over_time=same)
    grads = torch.autograd.grad(y, (x, r) if residual else (x,), dy)
    factors = ref.keep_factors(shape, p, seed, offset, same)
    check(y, x, factors, r)
    check(grads[0], dy, factors)
    if residual:
        assert torch.equal(grads[1], dy)


SHAPES = [(1,), (7,), (8,), (9,), (1023,), (2, 3, 5), (5, 3, 8), (4, 2, 129), (3, 7, 64), (13, 1, 333), (1, 1, 4099), (6, 2, 3, 11)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(shape, dtype):
    for p, residual, same in ((0.1, False, False), (0.5, True, False), (0.3, False, True), (0.9, True, True)):
        announce("dropout", shape, dtype, p, residual, same)
        run(shape, dtype, p, residual=residual, same=same)


@pytest.mark.parametrize("seed,offset", [(0, 0), (2**64 - 1, 2**64 - 1), (1 << 32, 1 << 32), (3, 2**32 - 1)])
def test_all_words_of_seed_and_offset_count(seed, offset):
    announce("dropout words", seed, offset)
    run((40, 33), "f32", 0.5, seed=seed, offset=offset)


def test_probabilities_at_the_ends():
    announce("dropout ends")
    x = torch.randn((3, 1000), device=DEV)
    assert torch.equal(dropout(x, 0.0, seed=1), x)
    assert not dropout(x, 1.0, seed=1).any()
    r = torch.randn_like(x)
    assert torch.equal(dropout(x, 1.0, seed=1, residual=r), r)
    # the smallest and the largest probability that drop and keep something
    keep = ref.draws(0, 3000, 1, 0)
    assert torch.equal((dropout(x, 1e-9, seed=1) != 0).cpu().flatten(), torch.from_numpy(keep >= 1) & (x != 0).cpu().flatten())
    assert torch.equal((dropout(x, 1 - 1e-9, seed=1) != 0).cpu().flatten(), torch.from_numpy(keep >= 65535) & (x != 0).cpu().flatten())


def test_what_is_dropped_is_not_multiplied():
    """Infinities and NaN in dropped places do not come through, in kept ones they do; nor in the gradient."""
    announce("dropout nan")
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.full((3, 100), bad, device=DEV, requires_grad=True)
        y = dropout(x, 0.5, seed=9)
        keep = torch.from_numpy(ref.keep_factors((3, 100), 0.5, 9, 0) != 0).to(DEV)
        assert not y[~keep].any() and not torch.isfinite(y[keep]).any()
        (dx,) = torch.autograd.grad(y, x, x.detach())
        assert not dx[~keep].any() and not torch.isfinite(dx[keep]).any()


def test_the_mask_is_that_of_the_index():
    """Whatever the type, the pitch, the order and the alignment of what it is applied to."""
    announce("dropout layouts")
    T, B, n, p, seed = 6, 5, 40, 0.4, 77
    x = torch.randn((T, B, n), device=DEV)
    for same in (False, True):
        want = dropout(x, p, seed=seed, same_over_time=same)
        assert torch.equal(dropout(x.bfloat16(), p, seed=seed, same_over_time=same) != 0, want != 0)
        for at, width in ((0, n + 8), (1, n + 1), (3, n + 17), (8, n + 8)):
            wide = torch.full((T, B, width), float("nan"), device=DEV)
            wide[..., at : at + n] = x if at + n <= width else 0
            if at + n > width:
                continue
            view = wide[..., at : at + n]
            assert torch.equal(dropout(view, p, seed=seed, same_over_time=same), want)
            assert torch.equal(dropout(x, p, seed=seed, same_over_time=same, residual=view), dropout(x, p, seed=seed, same_over_time=same, residual=x))
            assert torch.equal(dropout(view, p, seed=seed, same_over_time=same, residual=view), dropout(x, p, seed=seed, same_over_time=same, residual=x))
        other = x.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(dropout(other, p, seed=seed, same_over_time=same), want)
        flat = torch.empty((T * B * n + 3,), device=DEV)
        for at in (1, 2, 3):
            odd = flat[at : at + T * B * n].view(T, B, n)
            odd.copy_(x)
            assert torch.equal(dropout(odd, p, seed=seed, same_over_time=same), want)
        one = x[:1].expand(T, B, n)
        assert torch.equal(dropout(one, p, seed=seed, same_over_time=True)[0], dropout(one, p, seed=seed, same_over_time=True)[T - 1])
    leaf = x.clone().requires_grad_()
    dropout(leaf, p, seed=seed).sum().backward()  # an expanded error
    check(leaf.grad, torch.ones_like(x), ref.keep_factors((T, B, n), p, seed, 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,n", [(1, 3), (2, 9)])
def test_many_frames_share_a_mask(B, n, dtype):
    """More of them than a grid has rows, in one piece and with a pitch."""
    announce("dropout many frames", B, n, dtype)
    T, p, seed = 70001, 0.4, 21
    wide = torch.randn((T, B, n + 2), device=DEV).to(_DTYPES[dtype])
    factors = torch.from_numpy(ref.keep_factors((1, B, n), p, seed, 0, True).copy()).to(DEV)
    for x in (wide[..., :n], wide[..., :n].contiguous()):
        for r in (None, wide[..., 1 : n + 1]):
            y = dropout(x, p, seed=seed, residual=r, same_over_time=True)
            want = x.double() * factors + (0.0 if r is None else r.double())
            size = (x.double() * factors).abs() + (0.0 if r is None else r.double().abs())
            half = 2.0**-8 if dtype == "bf16" else U
            assert torch.all((y.double() - want).abs() <= 4 * U * size + half * want.abs())


def test_empty_and_refusals():
    announce("dropout refusals")
    for shape in ((0,), (0, 3), (3, 0), (2, 0, 4)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = dropout(x, 0.5, seed=1, same_over_time=len(shape) > 1)
        assert y.shape == x.shape
        y.sum().backward()
    x = torch.zeros((3, 4), device=DEV)
    for bad in (dict(residual=x[:2]), dict(residual=x.bfloat16()), dict(residual=torch.zeros((3, 4))), dict(offset=torch.zeros((1,), dtype=torch.int64)),
                dict(offset=torch.zeros((2,), dtype=torch.int64, device=DEV)), dict(offset=torch.zeros((1,), device=DEV))):  # fmt: skip
        with pytest.raises(RuntimeError):
            dropout(x, 0.5, seed=1, **bad)
    for t in (x.half(), x.double(), x.long(), torch.zeros((), device=DEV)):
        with pytest.raises(RuntimeError):
            dropout(t, 0.5, seed=1)
    with pytest.raises(RuntimeError, match="gradient"):
        leaf = x.clone().requires_grad_()
        torch.autograd.grad(dropout(leaf, 0.5, seed=1).sum(), leaf, create_graph=True)


@pytest.mark.parametrize("same", [False, True])
def test_beyond_32_bits(same):
    """Elements past 2^31 and groups at the end of the range of the index."""
    announce("dropout beyond 32 bits", same)
    shape = (3, (1 << 30) + 3) if not same else (2, (1 << 31) + 5)
    x = torch.ones(shape, dtype=torch.bfloat16, device=DEV)
    y = dropout(x, 0.5, seed=21, offset=1 << 40, same_over_time=same)
    width = shape[1]
    for row in range(shape[0]):
        for first in (0, width // 2 - 11, width - 40):
            e = first if same else row * width + first
            keep = ref.draws(e, 40, 21, 1 << 40) >= 32768
            assert numpy.array_equal(array(y[row, first : first + 40]), keep * 2.0)


def test_module_draws_anew_and_repeats():
    announce("dropout module")
    m = Dropout(0.5, seed=3)
    x = torch.ones((4, 64), device=DEV)
    a, b = m(x), m(x, residual=x)
    assert not torch.equal(a, b - x) and m.offset == 2
    m.offset = 0
    assert torch.equal(m(x), a) and torch.equal(m(x, residual=x), b)


def test_recorded_calls_draw_anew():
    """The offset on the device: forward and gradient of every replay take the one that lies there."""
    announce("dropout capture")
    x = torch.randn((5, 3, 130), device=DEV, requires_grad=True)
    dy = torch.randn((5, 3, 130), device=DEV)
    offset = torch.zeros((1,), dtype=torch.int64, device=DEV)

    def step():
        y = dropout(x, 0.3, seed=8, offset=offset)
        return (y.detach(),) + torch.autograd.grad(y, x, dy)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        offset += 1
    for k in range(4):
        offset.fill_(10 * k)
        graph.replay()
        torch.cuda.synchronize()
        y = dropout(x, 0.3, seed=8, offset=10 * k)
        want = (y,) + torch.autograd.grad(y, x, dy)
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        assert int(offset) == 10 * k + 1


def test_an_offset_changed_before_the_backward_pass_is_found():
    announce("dropout offset changed")
    x = torch.randn((5, 130), device=DEV, requires_grad=True)
    offset = torch.zeros((1,), dtype=torch.int64, device=DEV)
    y = dropout(x, 0.3, seed=8, offset=offset)
    offset += 1
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()
