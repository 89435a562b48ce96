"""The gated delta rule and its gradient against its definition in float64, on cuda:0."""

from __future__ import annotations

import numpy
import pytest
import torch

import _model_ref as ref
from _gpu_util import announce
from returnn_amd.delta_rule import DeltaRecurrence, gated_delta_rule

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = ("y", "s", "dq", "dk", "dv", "dg", "db", "ds0")


def inputs(T, B, Hk, H, dk, dv, dtype, seed=1, *, state=True, decay=1.0, strength=None):
    """Queries and keys of length 1 (or a little less), decays of which some are large, write strengths in [0,1]."""
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn((T, B, Hk, dk), generator=gen, dtype=torch.float64) for _ in range(2))
    q, k = (0.99 * t / t.norm(dim=-1, keepdim=True).clamp(min=1e-3) for t in (q, k))
    v = torch.randn((T, B, H, dv), generator=gen, dtype=torch.float64)
    g = -decay * torch.nn.functional.softplus(2 * torch.randn((T, B, H), generator=gen, dtype=torch.float64) - 3)
    b = torch.rand((T, B, H), generator=gen, dtype=torch.float64) if strength is None else torch.full((T, B, H), strength, dtype=torch.float64)
    s0 = torch.randn((B, H, dk, dv), generator=gen, dtype=torch.float64) if state else None
    dy, ds = torch.randn((T, B, H, dv), generator=gen, dtype=torch.float64), torch.randn((B, H, dk, dv), generator=gen, dtype=torch.float64)
    cast = [t.to(dtype).to(DEV) for t in (q, k, v)] + [t.float().to(DEV) for t in (g, b)] + [None if s0 is None else s0.float().to(DEV)]
    return cast, dy.to(dtype).to(DEV), ds.float().to(DEV)


def numbers(t):
    return None if t is None else t.detach().double().cpu().numpy()


def tolerances(dtype, names, want, terms):
    """
    Every result is made of sums of up to `terms` products (dk or dv of them, and 64 of a chunk, one after the other), each good to 2^-23 of the largest: of values about as large as the
    result's largest, `terms` of them are off by terms 2^-23 of it at most.  What ends in bfloat16 is rounded once (2^-8 of itself at most), and made of products of two parts
    (16 bits of each number: 2^-15 of the largest for sums of either sign).
    """
    for name, w in zip(names, want):
        most = abs(w).max(initial=0.0)
        if dtype == torch.bfloat16 and name in ("y", "dq", "dk", "dv"):
            yield 2.0**-8 * abs(w) + (terms * 2.0**-23 + 2.0**-11) * most + 1e-30
        else:
            yield terms * 2.0**-23 * most + 1e-30


def check(x, dy, ds, *, lens=None, direction=1, train=True, scale=None, terms=None):
    T, B, H, dv = x[2].shape
    dk = x[0].shape[-1]
    leaves = [t if t is None else t.clone().requires_grad_(train) for t in x]
    y, s = gated_delta_rule(*leaves[:5], state=leaves[5], seq_lens=None if lens is None else torch.tensor(lens), direction=direction, scale=scale)
    assert y.dtype == x[2].dtype and s.dtype == torch.float32 and y.shape == x[2].shape and s.shape == (B, H, dk, dv)
    a = [numbers(t) for t in x]
    want = list(ref.delta(*a, lens, direction, scale)[:2])
    got = [y, s]
    if train:
        given = [t for t in leaves if t is not None]
        got += torch.autograd.grad((y, s), given, (dy, ds))
        want += ref.delta_grad(*a[:5], numbers(dy), numbers(ds), a[5], lens, direction, scale)[: len(given)]
        for t, d in zip(given, got[2:]):
            assert d.dtype == t.dtype and d.shape == t.shape
    got = [numbers(t) for t in got]
    terms = terms or max(dk, dv) + 4 * 64
    for name, g, w, tol in zip(NAMES, got, want, tolerances(x[2].dtype, NAMES, want, terms)):
        off = abs(g - w)
        assert (off <= tol).all(), (name, off.max(), (off / tol).max())
    if lens is not None:
        past = numpy.arange(T)[:, None] >= numpy.clip(lens, 0, T)[None, :]
        for name, g in zip(NAMES, got):
            if name not in ("s", "ds0"):
                assert not g[past].any(), name
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 128, 129, 200])
def test_lengths(T, dtype):
    announce("delta lengths", T, dtype)
    x, dy, ds = inputs(T, 2, 1, 2, 24, 20, dtype, seed=T)
    check(x, dy, ds, train=False)
    check(x, dy, ds)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (7, 8), (8, 7), (16, 9), (31, 33), (32, 16), (33, 15), (40, 64), (64, 65), (65, 3), (100, 71), (127, 130), (128, 128), (128, 200)])
def test_widths(dk, dv, dtype):
    announce("delta widths", dk, dv, dtype)
    x, dy, ds = inputs(70, 2, 2, 2, dk, dv, dtype, seed=dk + 1000 * dv)
    check(x, dy, ds, direction=-1)
    check([t if t is None else t[:3] if t.dim() < 4 or t.shape[0] == 70 else t for t in x], dy, ds, train=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("direction", [1, -1])
@pytest.mark.parametrize("T", [9, 100])
def test_ragged(T, direction, dtype):
    """Lengths of 0, 1 and beyond T; what lies past a sequence's end is not read."""
    announce("delta ragged", T, direction, dtype)
    lens = [T, 0, 1, T // 2 + 1, T + 5, -3]
    x, dy, ds = inputs(T, 6, 2, 4, 17, 19, dtype, seed=T)
    past = (torch.arange(T)[:, None] >= torch.tensor(lens)[None, :]).to(DEV)
    for t in x[:5] + [dy]:
        t[past] = float("nan")
    check(x, dy, ds, lens=lens, direction=direction, train=False)
    got = check(x, dy, ds, lens=lens, direction=direction)
    assert numpy.array_equal(got[1][[1, 5]], numbers(x[5])[[1, 5]]) and numpy.array_equal(got[7][[1, 5]], numbers(ds)[[1, 5]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T,B,heads,dk,dv,lens", [(1500, 1, 1, 32, 40, None), (900, 2, 2, 128, 16, [900, 310]), (2200, 2, 1, 64, 130, [1, 2200])])
def test_segments(T, B, heads, dk, dv, lens, dtype):
    """Few sequences and heads: chunks in segments, of which a sequence may have none."""
    announce("delta segments", T, B, heads, dk, dv, dtype)
    x, dy, ds = inputs(T, B, heads, heads, dk, dv, dtype, seed=T, decay=0.05)
    check(x, dy, ds, lens=lens, train=False)
    check(x, dy, ds, lens=lens)
    check(x, dy, ds, lens=lens, direction=-1)


@pytest.mark.parametrize("key_heads,heads", [(1, 1), (1, 4), (2, 6), (3, 3), (5, 10)])
def test_shared_heads(key_heads, heads):
    announce("delta heads", key_heads, heads)
    for dtype in (torch.float32, torch.bfloat16):
        x, dy, ds = inputs(80, 2, key_heads, heads, 16, 24, dtype, seed=heads)
        check(x, dy, ds)
        check([t[:2] if t.dim() != 4 or t.shape[0] == 80 else t for t in x], dy, ds, train=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_decays_and_strengths_at_their_ends(dtype):
    """No decay, all forgotten (log decay of minus infinity and of the type's lowest value), nothing written, all replaced, more than that."""
    announce("delta extremes", dtype)
    for strength in (0.0, 1.0, 2.0):
        x, dy, ds = inputs(90, 2, 1, 2, 20, 12, dtype, seed=3, strength=strength)
        x[3][:, 0] = 0.0
        check(x, dy, ds, terms=4000)
    x, dy, ds = inputs(90, 2, 1, 2, 20, 12, dtype, seed=4)
    x[4][::3] = 0.0
    x[3][40, 0], x[3][41, 1], x[3][64, 0], x[3][::7, 1, 1] = -numpy.inf, torch.finfo(torch.float32).min, -numpy.inf, -1000.0
    check(x, dy, ds)
    check([t[38:45] if t.shape[0] == 90 else t for t in x], dy, ds, train=False)
    x[3].fill_(-numpy.inf)
    got = check(x, dy, ds)
    assert not got[7].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("B,H,dv", [(2, 2, 1), (1, 3, 40), (13, 10, 128)])
@pytest.mark.parametrize("T", [16, 128])
def test_large_states_that_cancel(T, B, H, dv, dtype):
    """
    A state a thousand times the values, of which a frame's write takes away just what its query asks for: key and query t are the unit vector t, so that y_t = scale (S_t + (v_t - S_t)).

    A chunk takes y_t from row t of the state before it, S (at most as large as s0 or v), and from u_t = v_t - S: together at most 2 |s0| + 3 |v|, no other number enters, and each is exact in three parts.
    So y is off by a few roundings to float32 of these, of which 10 of 2^-23 are allowed (products, their sums part by part, scale), and its own rounding.  A third part left out would be up to 2^-17.
    dq_t likewise, with an error dy_t of one column: element i from row i of S and from u_i where a frame i has written it.
    """
    announce("delta cancelling", T, B, H, dv, dtype)
    x, dy, ds = inputs(T, B, H, H, 128, dv, dtype, seed=21)
    unit = torch.eye(128, device=DEV, dtype=dtype)[:T, None, None, :].expand(T, B, H, 128)
    x[0], x[1], x[5] = unit.clone(), unit.clone(), 1000 * x[5]
    x[3].zero_()
    x[4].fill_(1.0)
    dy = dy * torch.eye(dv, device=DEV, dtype=dtype)[torch.arange(T) % dv][:, None, None, :]
    leaves = [t.clone().requires_grad_() for t in x]
    y, s = gated_delta_rule(*leaves[:5], state=leaves[5])
    (dq,) = torch.autograd.grad(y, leaves[0], dy)
    with torch.no_grad():
        z, r = gated_delta_rule(*x[:5], state=x[5])
    a = [numbers(t) for t in x]
    scale, e = 128**-0.5, abs(numbers(dy))
    want, state, _ = ref.delta(*a)
    want_q = ref.delta_grad(*a[:5], numbers(dy), numpy.zeros_like(a[5]), a[5])[0]
    half = torch.finfo(dtype).eps / 2
    parts = 2 * abs(a[5])
    parts[:, :, :T] += 3 * abs(a[2]).transpose(1, 2, 0, 3)
    for t in range(T):
        tol = half * abs(want[t]) + 10 * 2.0**-23 * scale * parts[:, :, t]
        for got in (y, z):
            off = abs(numbers(got[t]) - want[t])
            assert (off <= tol).all(), ("y", t, (off / tol).max())
        tol = half * abs(want_q[t]) + 10 * 2.0**-23 * scale * numpy.einsum("bhij,bhj->bhi", parts, e[t]) + 1e-30
        off = abs(numbers(dq[t]) - want_q[t])
        assert (off <= tol).all(), ("dq", t, (off / tol).max())
    for got in (s, r):
        assert (abs(numbers(got) - state) <= 8 * 2.0**-24 * abs(a[5]).max()).all()


def test_equal_keys():
    """The same key at every frame, written at full strength without decay: each value replaces the one before it; the inverse's entries are 1 and -1."""
    announce("delta equal keys")
    x, dy, ds = inputs(130, 1, 1, 1, 8, 16, torch.float32, seed=5, strength=1.0)
    x[1][:] = 0.0
    x[1][..., 2] = 1.0
    x[3].zero_()
    y, s = gated_delta_rule(*x[:5], state=x[5])
    assert (s[0, 0, 2] - x[2][-1, 0, 0]).abs().max() <= 130 * 2.0**-23 * 4
    check(x, dy, ds)


def test_no_state_scale_and_types():
    announce("delta optional arguments")
    x, dy, ds = inputs(50, 2, 2, 2, 16, 16, torch.float32, state=False)
    check(x, dy, ds, scale=2.5)
    y, s = gated_delta_rule(*x[:5])
    z, r = gated_delta_rule(*x[:5], state=torch.zeros((2, 2, 16, 16), device=DEV), scale=0.25, seq_lens=torch.tensor([50, 50], dtype=torch.int32, device=DEV))
    assert torch.equal(y, z) and torch.equal(s, r)
    g16 = x[3].bfloat16()
    y, s = gated_delta_rule(x[0], x[1], x[2], g16, x[4].double())
    z, r = gated_delta_rule(x[0], x[1], x[2], g16.float(), x[4])
    assert torch.equal(y, z) and torch.equal(s, r)
    leaf = g16.requires_grad_()
    (d,) = torch.autograd.grad(gated_delta_rule(x[0], x[1], x[2], leaf, x[4])[0].sum(), leaf)
    assert d.dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_steps_are_the_sequence(dtype):
    """Frame by frame with the state handed on, in short pieces, and all at once."""
    announce("delta steps", dtype)
    T = 40
    x, _, _ = inputs(T, 3, 2, 4, 24, 30, dtype, seed=9)
    y, s = gated_delta_rule(*x[:5], state=x[5])
    for piece in (1, 7, 16):
        state, ys = x[5], []
        for t in range(0, T, piece):
            part = [a[t] if piece == 1 else a[t : t + piece] for a in x[:5]]
            z, state = gated_delta_rule(*part, state=state)
            ys.append(z[None] if piece == 1 else z)
        # (both sides good to what `tolerances` says)
        most = float(y.abs().max()), float(s.abs().max())
        assert (torch.cat(ys).float() - y.float()).abs().max() <= (2.0**-7 + 2.0**-10 if dtype == torch.bfloat16 else 2 * 300 * 2.0**-23) * most[0]
        assert (state - s).abs().max() <= 2 * 300 * 2.0**-23 * most[1]


def test_slices_of_a_projection():
    """Queries, keys and values as parts of rows with a pitch, an error with one, and tensors in another order."""
    announce("delta slices")
    T, B, Hk, H, dk, dv = 70, 3, 2, 2, 20, 33
    for dtype in (torch.float32, torch.bfloat16):
        x, dy, ds = inputs(T, B, Hk, H, dk, dv, dtype, seed=11)
        row = torch.cat([t.flatten(2) for t in x[:3]] + [torch.zeros((T, B, 5), dtype=dtype, device=DEV)], dim=-1).requires_grad_()
        q, k, v, _ = row.split([Hk * dk, Hk * dk, H * dv, 5], dim=-1)
        parts = q.unflatten(-1, (Hk, dk)), k.unflatten(-1, (Hk, dk)), v.unflatten(-1, (H, dv))
        y, s = gated_delta_rule(*parts, *x[3:5], state=x[5])
        wide = torch.zeros((T, B, H * dv + 3), dtype=dtype, device=DEV)
        wide[..., : H * dv] = dy.flatten(2)
        got = torch.autograd.grad((y, s), row, (wide[..., : H * dv].unflatten(-1, (H, dv)), ds))[0]
        leaves = [t.clone().requires_grad_() for t in x[:3]]
        z, r = gated_delta_rule(*leaves, *x[3:5], state=x[5])
        want = torch.autograd.grad((z, r), leaves, (dy, ds))
        assert torch.equal(y, z) and torch.equal(s, r)
        for g, w in zip(got.split([Hk * dk, Hk * dk, H * dv, 5], dim=-1), want):
            assert torch.equal(g, w.flatten(2))
        turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in x[:5]]
        z, r = gated_delta_rule(*turned, state=x[5].transpose(2, 3).contiguous().transpose(2, 3))
        assert torch.equal(y, z) and torch.equal(s, r)


def test_repeated_calls_agree():
    announce("delta repeated")
    x, dy, ds = inputs(300, 2, 2, 4, 64, 128, torch.bfloat16, seed=12)
    leaves = [t.clone().requires_grad_() for t in x]
    runs = []
    for _ in range(3):
        y, s = gated_delta_rule(*leaves[:5], state=leaves[5], seq_lens=torch.tensor([300, 170]))
        runs.append((y, s) + torch.autograd.grad((y, s), leaves, (dy, ds)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_parts_of_the_gradient():
    """Only the output's error, only the state's, only some of the inputs."""
    announce("delta partial gradients")
    x, dy, ds = inputs(66, 2, 1, 2, 16, 16, torch.float32, seed=13)
    leaves = [t.clone().requires_grad_() for t in x]
    y, s = gated_delta_rule(*leaves[:5], state=leaves[5])
    both = torch.autograd.grad((y, s), leaves, (dy, ds), retain_graph=True)
    one, other = (torch.autograd.grad(t, leaves, e, retain_graph=True) for t, e in ((y, dy), (s, ds)))
    for a, b, c in zip(both, one, other):
        assert (a - b - c).abs().max() <= 3 * 300 * 2.0**-23 * max(float(t.abs().max()) for t in (a, b, c))
    y, s = gated_delta_rule(x[0], x[1], leaves[2], x[3], x[4])
    (dv,) = torch.autograd.grad(y, leaves[2], dy)
    assert dv.abs().max() > 0
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(gated_delta_rule(*leaves[:5])[0].sum(), leaves[0], create_graph=True)


def test_another_stream_and_recorded_steps():
    """On a stream of its own; recorded into a graph, forward and gradient, and replayed with other inputs and eager work between."""
    announce("delta streams and graphs")
    T, B, H, dk, dv = 200, 1, 2, 32, 48
    x, dy, ds = inputs(T, B, H, H, dk, dv, torch.bfloat16, seed=14)
    lens = torch.tensor([150], device=DEV)

    def step(leaves):
        y, s = gated_delta_rule(*leaves[:5], state=leaves[5], seq_lens=lens)
        return (y, s) + torch.autograd.grad((y, s), leaves, (dy, ds))

    def fresh(of):
        return [t.clone().requires_grad_() for t in of]

    want = step(fresh(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(fresh(x))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    static = fresh(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)  # (warm-up on the capture's side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step(static)
    for seed in (14, 15, 16):
        other, _, _ = inputs(T, B, H, H, dk, dv, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for a, b in zip(static, other):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(fresh(other))
        assert all(torch.equal(a, b) for a, b in zip(want, recorded)), seed


def test_empty():
    announce("delta empty")
    g = torch.zeros((0, 2, 3), device=DEV)
    s0 = torch.randn((2, 3, 4, 5), device=DEV).requires_grad_()
    y, s = gated_delta_rule(torch.zeros((0, 2, 3, 4), device=DEV), torch.zeros((0, 2, 3, 4), device=DEV), torch.zeros((0, 2, 3, 5), device=DEV), g, g, state=s0)
    assert y.shape == (0, 2, 3, 5) and torch.equal(s, s0)
    assert torch.equal(torch.autograd.grad(s.sum(), s0)[0], torch.ones_like(s0))
    for B, H in ((0, 3), (2, 0)):
        y, s = gated_delta_rule(*(torch.zeros((6, B, H, n), device=DEV) for n in (4, 4, 5)), torch.zeros((6, B, H), device=DEV), torch.zeros((6, B, H), device=DEV))
        assert y.shape == (6, B, H, 5) and s.shape == (B, H, 4, 5)


def bf16_bound(got, want, terms):
    """As `tolerances`, but with all numbers in three parts: what ends in bfloat16 is off by its own rounding and as float32 results are."""
    for name, g, w in zip(NAMES, got, want):
        most = abs(w).max(initial=0.0)
        tol = (2.0**-8 * abs(w) if name in ("y", "dq", "dk", "dv") else 0.0) + terms * 2.0**-23 * most + 1e-30
        off = abs(g - w)
        assert (off <= tol).all(), (name, off.max(), (off / tol).max())


@pytest.mark.parametrize("T,B,Hk,H,dk,dv,direction,lens", [
    (17, 2, 1, 2, 24, 20, 1, None), (100, 6, 2, 4, 17, 19, -1, [100, 0, 1, 51, 105, -3]), (200, 2, 2, 2, 128, 130, 1, None), (70, 2, 2, 2, 65, 3, -1, None),
    (900, 2, 2, 2, 128, 16, 1, [900, 310]), (2200, 2, 1, 1, 64, 130, -1, [1, 2200]),
])  # fmt: skip
def test_bfloat16_is_rounded_once(T, B, Hk, H, dk, dv, direction, lens):
    """Short, ragged, wide and narrow calls and such in segments against the bound that has no place for a part left out."""
    announce("delta rounded once", T, B, Hk, H, dk, dv, direction)
    x, dy, ds = inputs(T, B, Hk, H, dk, dv, torch.bfloat16, seed=T + dv, decay=0.05 if T > 200 else 1.0)
    got = check(x, dy, ds, lens=lens, direction=direction)
    a = [numbers(t) for t in x]
    want = list(ref.delta(*a, lens, direction)[:2]) + list(ref.delta_grad(*a[:5], numbers(dy), numbers(ds), a[5], lens, direction))
    bf16_bound(got, want, max(dk, dv) + 4 * 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("Hk,dk,dv,direction", [(3, 20, 128, 1), (1, 40, 71, -1), (3, 128, 128, -1), (1, 128, 100, 1)])
def test_many_heads(Hk, dk, dv, direction, dtype):
    """129 heads of more than 64 columns: eight wavefronts a workgroup, of several widths, ragged, with shared queries and keys."""
    announce("delta many heads", Hk, dk, dv, direction, dtype)
    T, B, H = 70, 43, 3
    x, dy, ds = inputs(T, B, Hk, H, dk, dv, dtype, seed=dk + dv)
    lens = [T - n % 9 * 7 for n in range(B)]
    lens[3:5] = 0, 1
    got = check(x, dy, ds, lens=lens, direction=direction)
    a = [numbers(t) for t in x]
    want = list(ref.delta(*a, lens, direction)[:2]) + list(ref.delta_grad(*a[:5], numbers(dy), numbers(ds), a[5], lens, direction))
    if dtype == torch.bfloat16:
        bf16_bound(got, want, max(dk, dv) + 4 * 64)
    y, s = gated_delta_rule(*x[:5], state=x[5], seq_lens=torch.tensor(lens), direction=direction)  # (no gradient follows)
    assert numpy.array_equal(numbers(y), got[0]) and numpy.array_equal(numbers(s), got[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_shared_heads_in_segments(dtype):
    announce("delta shared heads in segments", dtype)
    x, dy, ds = inputs(1100, 2, 2, 6, 40, 24, dtype, seed=8, decay=0.05)
    for direction in (1, -1):
        check(x, dy, ds, lens=[1100, 700], direction=direction)


def test_no_heads_of_values():
    """Queries and keys of heads that have no values: their gradient is zero."""
    announce("delta no values")
    for dtype in (torch.float32, torch.bfloat16):
        for T in (1, 6, 70):
            q, k = (torch.ones((T, 2, 3, 24), device=DEV, dtype=dtype, requires_grad=True) for _ in "qk")
            v, g = torch.zeros((T, 2, 0, 5), device=DEV, dtype=dtype), torch.zeros((T, 2, 0), device=DEV)
            y, s = gated_delta_rule(q, k, v, g, g)
            assert y.shape == (T, 2, 0, 5) and s.shape == (2, 0, 24, 5)
            used = [torch.full_like(q, float("nan")) for _ in range(4)]
            del used  # (what memory holds that is given out next)
            for d in torch.autograd.grad(y.sum() + s.sum(), [q, k]):
                assert torch.equal(d, torch.zeros_like(q))


def test_refusals():
    announce("delta refusals")
    x, _, _ = inputs(5, 2, 2, 4, 8, 6, torch.float32)
    q, k, v, g, b, s0 = x

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            gated_delta_rule(*args, **kw)

    refused("match", q, k[:, :1], v, g, b)
    refused("match", q[0], k[0], v, g, b)
    refused("one type", q.bfloat16(), k, v, g, b)
    refused("float32 or bfloat16", q.half(), k.half(), v.half(), g, b)
    refused("evenly", q, k, v[:, :, :3], g[:, :, :3], b[:, :, :3])
    refused("log_decay", q, k, v, g[:, :, :2], b)
    refused("beta", q, k, v, g, b.long())
    refused("state", q, k, v, g, b, state=s0[:1])
    refused("seq_lens", q, k, v, g, b, seq_lens=torch.tensor([1]))
    refused("seq_lens", q, k, v, g, b, seq_lens=torch.tensor([1.0, 2.0]))
    refused("direction", q, k, v, g, b, direction=0)
    refused("elements needed", torch.zeros((5, 2, 2, 129), device=DEV), torch.zeros((5, 2, 2, 129), device=DEV), v, g, b)
    refused("is on", q, k, v, g.cpu(), b)
    refused("values must be", q[0, 0], k[0, 0], v[0, 0], g[0, 0], b[0, 0])
    with torch.autograd.forward_ad.dual_level():
        refused("forward mode", q, k, torch.autograd.forward_ad.make_dual(v, v), g, b)
    with torch.autocast("cuda", dtype=torch.float16):
        y, _ = gated_delta_rule(q.half(), k.half(), v.half(), g, b)
    assert y.dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_layer(dtype):
    """The layer against its own definition; in a region of autocast; single steps."""
    announce("delta layer", dtype)
    torch.manual_seed(2)
    m = DeltaRecurrence(20, 64, num_heads=2, key_dim=24, device=DEV, dtype=dtype)
    x = torch.randn((70, 3, 20), device=DEV, dtype=dtype)
    y, s = m(x, seq_lens=torch.tensor([70, 5, 33]))
    assert y.shape == (70, 3, 64) and y.dtype == dtype and s.shape == (3, 2, 24, 32)
    q, k, v, g, b = torch.nn.functional.linear(x, m.ff, m.bias).split(m.split, dim=-1)
    q, k = (m._unit(t.unflatten(-1, (2, 24))) for t in (q, k))
    assert (k.float().norm(dim=-1) < 1 + 2.0**-7).all()
    want, state, _ = ref.delta(*(numbers(t) for t in (q, k, v.unflatten(-1, (2, 32)), -torch.nn.functional.softplus(g.float()), torch.sigmoid(b.float()))), lens=[70, 5, 33])
    tol = list(tolerances(dtype, ("y", "s"), (want.reshape(70, 3, 64), state), 300))
    assert (abs(numbers(y) - want.reshape(70, 3, 64)) <= tol[0]).all() and (abs(numbers(s) - state) <= tol[1]).all()
    y.float().sum().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in m.parameters())
    z, r = m(x[0])
    assert z.shape == (3, 64) and (z - y[0]).abs().max() <= 2.0**-6 * float(y.detach().abs().max())
    if dtype == torch.float32:
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert m(x)[0].dtype == torch.bfloat16


def test_offsets_beyond_32_bits():
    """States of more than 2^32 bytes kept for the gradient: a long call against its two halves, the state handed on."""
    announce("delta rule, long")
    T, half, B, H, d = 70000, 35008, 8, 8, 128
    gen = torch.Generator(device=DEV).manual_seed(12)
    q, k = (torch.nn.functional.normalize(torch.randn((T, B, H, d), device=DEV, generator=gen, dtype=torch.bfloat16), dim=-1) for _ in "qk")
    v, dy = (torch.randn((T, B, H, d), device=DEV, generator=gen, dtype=torch.bfloat16) for _ in "ve")
    g, b = -torch.rand((T, B, H), device=DEV, generator=gen) * 0.1, torch.rand((T, B, H), device=DEV, generator=gen)
    leaves = [t.requires_grad_() for t in (q, k, v, g, b)]
    y, s = gated_delta_rule(*leaves)
    whole = torch.autograd.grad(y, leaves, dy)
    state, parts = None, []
    for part in (slice(0, half), slice(half, T)):
        y1, state = gated_delta_rule(*(t[part] for t in leaves), state=state)
        parts.append(y1)
    chained = torch.autograd.grad(parts, leaves, [dy[:half], dy[half:]])
    assert (s - state).detach().norm() <= 1e-5 * s.detach().norm()
    # (two roundings to bfloat16 of numbers that agree to 1e-5)
    for a, c in [(y.detach(), torch.cat(parts).detach())] + list(zip(whole, chained)):
        for at in (slice(0, 2000), slice(half - 1000, half + 1000), slice(T - 2000, T)):
            x, z = a[at].float(), c[at].float()
            assert torch.isfinite(x).all() and (x - z).norm() <= (2.0**-7 if a.dtype == torch.bfloat16 else 1e-4) * x.norm()
