"""
Log probabilities, entropy, alternatives and their gradient on the GPU against their definitions in 64 bits.

Error bounds (u = 2^-24): an exponential of a difference d is good to (|d| + 8) u of itself, where it counts |d| is at most log V + 8; a
sum of V positive terms in at most V / 64 + 64 additions one after the other adds as many u.  So the logarithm of the sum is good to
S = (V / 64 + 2 log V + 96) u, a log probability to S + 4 u of its size, the entropy to 4 (1 + log V) S, and an element of the gradient to
4 S (2 + its |log p| + entropy) of the products it is made of.  bfloat16 gradients: 2^-8 of the value more.
The alternatives' indices are exact.
"""

from __future__ import annotations

import math

import numpy
import pytest
import torch

import _sequence_ref as ref
from _gpu_util import announce
from returnn_amd import lib, sequence_lib
from returnn_amd.scoring import token_log_probs

pytestmark = pytest.mark.gpu
U = 2.0**-24
DEV = "cuda:0"
INF = float("inf")
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def array(t):
    return t.detach().double().cpu().numpy()


def near(got, want, bound):
    """Equal where the definition is not finite, within the bound where it is."""
    finite = numpy.isfinite(want)
    assert numpy.array_equal(got[~finite], want[~finite], equal_nan=True)
    off = numpy.abs(got[finite] - want[finite])
    assert numpy.all(off <= numpy.broadcast_to(bound, want.shape)[finite]), (off.max(), numpy.max(bound))


def check(logits, targets, top_k, s, grads=None):
    x = array(logits).reshape(-1, logits.shape[-1])
    R, V = x.shape
    flat = None if targets is None else targets.reshape(-1).cpu().numpy()
    log_prob, entropy, top, ids, log_p = ref.scores(x, flat, top_k)
    S = (V / 64 + 2 * math.log(V) + 96) * U

    def size(a):
        return numpy.abs(numpy.nan_to_num(a, nan=0.0, posinf=0.0, neginf=0.0))

    if targets is not None:
        near(array(s.log_probs).reshape(R), log_prob, S + 4 * U * size(log_prob))
    else:
        assert s.log_probs is None
    if s.entropy is not None:
        near(array(s.entropy).reshape(R), entropy, 4 * (1 + math.log(V)) * S)
    assert s.top_log_probs.shape == logits.shape[:-1] + (top_k,) and s.top_ids.dtype == torch.int64
    assert numpy.array_equal(s.top_ids.reshape(R, top_k).cpu().numpy(), ids)
    near(array(s.top_log_probs).reshape(R, top_k), top, S + 4 * U * size(top))
    if grads is not None:
        g, ge, D = (None if t is None else array(t).reshape(R, -1) for t in grads)
        g = numpy.zeros((R, 1)) if g is None else g
        ge = numpy.zeros((R, 1)) if ge is None else ge
        want = ref.scores_grad(x, flat, g[:, 0], ge[:, 0])
        p = numpy.nan_to_num(numpy.exp(log_p))
        made_of = p * (numpy.abs(g) + numpy.abs(ge) * (size(log_p) + numpy.nan_to_num(entropy)[:, None]))
        if flat is not None:
            for r in range(R):
                if 0 <= flat[r] < V:
                    made_of[r, flat[r]] += abs(g[r, 0])
        half = 2.0**-8 if logits.dtype == torch.bfloat16 else U
        # (2^-126: what float32 cannot hold as a normal number)
        near(D, want, 4 * S * (2 + size(log_p) + numpy.nan_to_num(entropy)[:, None]) * made_of + half * size(want) + 2.0**-126)


def problem(rows, V, dtype, seed=0, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(tuple(rows) + (V,), generator=gen) * spread).to(_DTYPES[dtype])
    targets = torch.randint(0, V, tuple(rows), generator=gen)
    return logits, targets


def run(logits, targets, top_k, entropy=True, seed=1):
    leaf = logits.to(DEV).requires_grad_()
    td = None if targets is None else targets.to(DEV)
    s = token_log_probs(leaf, td, entropy=entropy, top_k=top_k)
    used = [t for t in (s.log_probs, s.entropy) if t is not None]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    errors = [torch.randn(t.shape, device=DEV, generator=gen) for t in used]
    D = torch.autograd.grad(used, leaf, errors)[0] if used else None
    by = dict(zip([n for n, t in (("g", s.log_probs), ("ge", s.entropy)) if t is not None], errors))
    plain = token_log_probs(leaf.detach(), td, entropy=entropy, top_k=top_k)
    for a, b in zip(s, plain):
        assert (a is None and b is None) or torch.equal(a, b) or torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    return s, (by.get("g"), by.get("ge"), D)


SHAPES = [((1,), 1), ((3,), 2), ((2, 2), 7), ((5,), 63), ((4,), 64), ((130,), 65), ((2, 3), 127), ((9,), 500), ((2,), 1023), ((3,), 1025), ((1,), 4096), ((2, 7), 2047), ((17,), 5003),
          ((1,), 10007), ((3,), 32000), ((1,), 131072), ((2,), 65537), ((600,), 33),
          ((700,), 200), ((3,), 8000), ((600,), 6001), ((1100,), 513), ((1100,), 1025)]  # fmt: skip


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", SHAPES)
def test_against_the_definition(rows, V, dtype):
    for k, given in ((0, True), (1, False), (min(V, 12), True), (min(V, 64), False)):
        announce("scores", rows, V, dtype, k, given)
        logits, targets = problem(rows, V, dtype, seed=V)
        targets = targets if given else None
        s, grads = run(logits, targets, k)
        check(logits, targets, k, s, grads)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_without_entropy_and_without_anything_but_alternatives(dtype):
    announce("scores parts", dtype)
    logits, targets = problem((6,), 700, dtype)
    s, grads = run(logits, targets, 3, entropy=False)
    assert s.entropy is None
    check(logits, targets, 3, s, grads)
    s, _ = run(logits, None, 5, entropy=False)
    check(logits, None, 5, s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 50, 1000, 20000, 70001])
def test_masked_logits(V, dtype):
    """Tokens that are not allowed: of minus infinity, of the type's lowest value; rows of nothing else; one token left."""
    announce("scores masked", V, dtype)
    lowest = torch.finfo(_DTYPES[dtype]).min
    logits, targets = problem((8,), V, dtype, seed=2)
    rng = torch.Generator().manual_seed(3)
    blocked = torch.rand((8, V), generator=rng) < 0.5
    logits[0][blocked[0]] = -INF
    logits[1][blocked[1]] = lowest
    logits[2] = -INF
    logits[3] = lowest
    logits[4] = -INF
    logits[4, V // 2] = 1.5
    logits[5][blocked[5]] = -INF
    logits[5, 0] = lowest
    logits[6] = lowest
    logits[6, V - 1] = 3.0
    targets[4] = V // 2
    targets[7] = -1
    logits[7] = float("nan")
    s, grads = run(logits, targets, min(V, 20))
    check(logits, targets, min(V, 20), s, grads)
    assert not grads[2][2].any() and not grads[2][7].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(9, 1), (9, 50), (300, 1000), (9, 5000), (300, 9001), (9, 20000), (9, 70001)])
def test_masked_logits_without_alternatives(rows, V, dtype):
    """The same, and masks of whole ranges of tokens, from the first one on; and values that are not finite."""
    announce("scores masked sums", rows, V, dtype)
    lowest = torch.finfo(_DTYPES[dtype]).min
    logits, targets = problem((rows,), V, dtype, seed=6)
    blocked = torch.rand((rows, V), generator=torch.Generator().manual_seed(5)) < 0.5
    logits[0][blocked[0]] = -INF
    logits[1][blocked[1]] = lowest
    logits[2] = -INF
    logits[3] = lowest
    logits[4, : V // 2] = -INF
    logits[5, : V - V // 3] = lowest
    logits[6, V // 4 :] = -INF
    logits[7] = -INF
    logits[7, V - 1] = -2.0
    logits[8, : V // 2] = lowest
    logits[8, V // 2 :] = -1e9
    s, grads = run(logits, targets, 0)
    check(logits, targets, 0, s, grads)
    for k, bad in enumerate((float("nan"), INF)):
        logits[k, V - 1 - k * (V // 3)] = bad
        logits[k + 2, (k + 1) * V // 4] = bad
    s, _ = run(logits, targets, 0)
    assert torch.isnan(s.log_probs[:4]).all() and torch.isnan(s.entropy[:4]).all() and not torch.isnan(s.entropy[4:]).any()


@pytest.mark.parametrize("V", [3, 90, 3000, 40000])
def test_not_finite_logits(V):
    """A NaN or an infinity makes its row NaN and no other; it comes first among the alternatives."""
    announce("scores nan", V)
    logits, targets = problem((5,), V, "f32", seed=4)
    logits[1, V // 2] = float("nan")
    logits[3, V - 1] = INF
    s, grads = run(logits, targets, 3)
    for r in (1, 3):
        assert torch.isnan(s.log_probs[r]) and torch.isnan(s.entropy[r]) and torch.isnan(grads[2][r]).all() and torch.isnan(s.top_log_probs[r]).all()
    assert int(s.top_ids[1, 0]) == V // 2 and int(s.top_ids[3, 0]) == V - 1
    rest = [0, 2, 4]
    check(logits[rest], targets[rest], 3, type(s)(*(t[rest] for t in s)), tuple(t[rest] for t in grads))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_targets_that_are_none(dtype):
    """Negative ones: rows that are not read (NaN lies there); too large ones: NaN in their rows alone."""
    announce("scores targets", dtype)
    for V in (33, 4100, 50000):
        logits, targets = problem((3, 4), V, dtype, seed=5)
        targets[0, 1], targets[2, 3] = -1, -(2**40)
        logits[0, 1] = float("nan")
        logits[2, 3] = float("nan")
        targets[1, 1], targets[1, 2] = V, 2**40
        s, grads = run(logits, targets, 2)
        check(logits, targets, 2, s, grads)
        assert not grads[2][0, 1].any() and torch.isnan(grads[2][1, 1]).all() and torch.isnan(grads[2][1, 2]).all()
        assert int(s.top_ids[0, 1, 0]) == -1 and float(s.log_probs[2, 3].detach()) == 0
        small = targets.to(torch.int32) if V < 2**31 and int(targets.max()) < 2**31 else targets.clamp(max=V)
        t = token_log_probs(logits.to(DEV), small.to(DEV), top_k=2)
        assert torch.equal(t.top_ids, s.top_ids)


@pytest.mark.parametrize("V", [64, 65, 1000, 32000, 100003])
def test_ties(V):
    """The lower index first: all equal, runs of equal ones, both zeros, ascending and descending rows."""
    announce("scores ties", V)
    for dtype in ("f32", "bf16"):
        logits = torch.zeros((8, V), dtype=_DTYPES[dtype])
        logits[0, ::2] = -0.0
        logits[1] = 1.0
        logits[2] = torch.arange(V).div(7, rounding_mode="floor").to(logits.dtype)
        logits[3] = -torch.arange(V).div(7, rounding_mode="floor").to(logits.dtype)
        logits[4, V // 3 :] = 2.0
        logits[5, V - 30 :] = 2.0
        logits[6] = torch.arange(V).to(logits.dtype)
        logits[7] = -torch.arange(V).to(logits.dtype)
        for k in (1, 10, 64):
            s = token_log_probs(logits.to(DEV), top_k=k)
            _, _, _, ids, _ = ref.scores(array(logits), None, k)
            assert numpy.array_equal(s.top_ids.cpu().numpy(), ids), (dtype, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [8, 9, 64, 100, 129, 256, 500, 513, 1000, 1025, 2048])
def test_many_short_rows(V, dtype):
    """Masks, ties and rows of nothing else, in more rows than have a workgroup each."""
    announce("scores many short rows", V, dtype)
    rows, lowest = 1201, torch.finfo(_DTYPES[dtype]).min
    logits, targets = problem((rows,), V, dtype, seed=8)
    blocked = torch.rand((rows, V), generator=torch.Generator().manual_seed(9)) < 0.5
    kind = torch.arange(rows) % 12
    logits[(kind == 0)[:, None] & blocked] = -INF
    logits[(kind == 1)[:, None] & blocked] = lowest
    logits[kind == 2] = -INF
    logits[kind == 3] = lowest
    logits[kind == 4] = 0.5
    logits[kind == 5] = torch.arange(V).div(7, rounding_mode="floor").to(logits.dtype)
    logits[kind == 6] = -torch.arange(V).to(logits.dtype)
    logits[kind == 7, V // 3 :] = 9.0
    logits[kind == 8, : V - 1] = -INF
    targets[kind == 9] = -1
    for k in (0, 1, 8, 16, 64):
        s, grads = run(logits, targets, min(k, V))
        check(logits, targets, min(k, V), s, grads)


@pytest.mark.parametrize("V,k", [(40000, 64), (65540, 33), (131072, 64), (500001, 7), (3000000, 64)])
def test_alternatives_of_rows_in_pieces(V, k):
    """Equal logits everywhere, or in one of the pieces, and best ones that all lie in one piece: ties go to the lower index."""
    announce("scores pieces", V, k)
    flat = torch.zeros((1, V), device=DEV)
    late = flat.clone()
    late[0, V - 100 : V - 100 + 2 * k : 2] = 1.0
    spread = flat.clone()
    spread[0, :: V // 50] = 2.0
    for logits in (flat, late, spread):
        s = token_log_probs(logits, top_k=k)
        want = torch.sort(logits[0].cpu(), descending=True, stable=True).indices[:k]
        assert torch.equal(s.top_ids[0].cpu(), want)
        # (a float32 result: the logarithm of a sum of 64-bit terms, and the sum's roundings, some units of 2^-24 each of up to 16)
        exact = torch.log_softmax(logits[0].double(), dim=-1)[s.top_ids[0]]
        assert (s.top_log_probs[0].double() - exact).abs().max() < 64 * 2.0**-24 * 16


def test_large_logits():
    """What a sum of one number for lse would round away: logits around 1e4, differences of a few."""
    announce("scores large")
    logits, targets = problem((6,), 300, "f32", seed=6)
    logits = (logits + torch.tensor([1e4, -1e4, 1e6, 3e37, -3e37, 0.0])[:, None]).contiguous()
    s, grads = run(logits, targets, 4)
    check(logits, targets, 4, s, grads)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_orders(dtype):
    """Vocabularies padded in the projection, rows at any address, other orders of the axes, expanded errors."""
    announce("scores strides", dtype)
    T, B, V = 5, 3, 1037
    logits, targets = problem((T, B), V, dtype, seed=7)
    ld, td = logits.to(DEV), targets.to(DEV)
    want = token_log_probs(ld, td, entropy=True, top_k=9)
    leaf = ld.clone().requires_grad_()
    (token_log_probs(leaf, td, entropy=True).log_probs.sum()).backward()
    for at, width in ((0, 1088), (1, 1038), (3, 1041), (8, 1064), (51, 1088)):
        wide = torch.full((T, B, width), float("nan"), dtype=ld.dtype, device=DEV)
        view = wide[..., at : at + V]
        view.copy_(ld)
        view = view.detach().requires_grad_()
        got = token_log_probs(view, td, entropy=True, top_k=9)
        check(logits, targets, 9, got)
        assert torch.equal(got.top_ids, want.top_ids)
        (d,) = torch.autograd.grad(got.log_probs.sum(), view)
        S = (V / 64 + 2 * math.log(V) + 96) * U
        assert d.shape == leaf.grad.shape and (d.float() - leaf.grad.float()).abs().max() <= 2.0**-8 * (dtype == "bf16") + 64 * S
    swapped = ld.transpose(0, 1).contiguous().transpose(0, 1)
    got = token_log_probs(swapped, td, entropy=True, top_k=9)
    assert torch.equal(got.log_probs, want.log_probs) and torch.equal(got.top_ids, want.top_ids)
    columns = ld.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # (the last axis is not the fastest)
    got = token_log_probs(columns, td.t().contiguous().t(), entropy=True, top_k=9)
    assert torch.equal(got.entropy, want.entropy) and torch.equal(got.log_probs, want.log_probs)
    one = token_log_probs(ld[0, 0], td[0, 0], entropy=True, top_k=9)  # a single row without leading axes
    assert one.log_probs.shape == () and torch.equal(one.top_ids, want.top_ids[0, 0])


def test_gradient_against_differences():
    """Of the definition's values, not of its gradient's formula."""
    announce("scores differences")
    R, V, h = 3, 11, 1e-5
    logits, targets = problem((R,), V, "f32", seed=8)
    targets[1] = -1
    s, (g, ge, D) = run(logits, targets, 0)
    x, g, ge = array(logits), array(g), array(ge)

    def value():
        lp, e, _, _, _ = ref.scores(x, targets.numpy())
        return (lp * g).sum() + (e * ge).sum()

    for at in numpy.ndindex(x.shape):
        old = x[at]
        x[at] = old + h
        up = value()
        x[at] = old - h
        down = value()
        x[at] = old
        assert abs((up - down) / (2 * h) - float(D[at])) < 1e-4  # (4 S (2 + 20 + 3) of products below 30)


def test_empty_and_refusals():
    announce("scores refusals")
    x = torch.zeros((0, 7), device=DEV, requires_grad=True)
    s = token_log_probs(x, torch.zeros((0,), dtype=torch.int64, device=DEV), entropy=True, top_k=3)
    assert s.log_probs.shape == (0,) and s.top_ids.shape == (0, 3)
    (s.log_probs.sum() + s.entropy.sum()).backward()
    x = torch.zeros((3, 7), device=DEV)
    t = torch.zeros((3,), dtype=torch.int64, device=DEV)
    for args, kw in (((x, t[:2]), {}), ((x, t.float()), {}), ((x, t.cpu()), {}), ((x, t), dict(top_k=8)), ((x, t), dict(top_k=-1)), ((x[:, :0], t), {}), ((x.half(), t), {}),
                     ((x.double(), t), {}), ((torch.zeros((2, 100), device=DEV),), dict(top_k=65))):  # fmt: skip
        with pytest.raises(RuntimeError):
            token_log_probs(*args, **kw)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        torch.autograd.grad(token_log_probs(leaf, t).log_probs.sum(), leaf, create_graph=True)
    s = token_log_probs(leaf, t, top_k=2)
    assert not s.top_log_probs.requires_grad
    torch.cuda.synchronize()


def test_beyond_32_bits():
    """Rows past 2^31 elements and 2^32 bytes, against the same rows by themselves."""
    announce("scores beyond 32 bits")
    R, V = 70001, 32001
    logits = torch.empty((R, V), dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1)).requires_grad_()
    targets = torch.randint(0, V, (R,), device=DEV)
    s = token_log_probs(logits, targets, entropy=True, top_k=2)
    (D,) = torch.autograd.grad(s.log_probs.sum() + s.entropy.sum(), logits)
    few = logits.detach()[-3:].clone().requires_grad_()
    f = token_log_probs(few, targets[-3:], entropy=True, top_k=2)
    (d,) = torch.autograd.grad(f.log_probs.sum() + f.entropy.sum(), few)
    check(few.detach().cpu(), targets[-3:].cpu(), 2, f)
    assert torch.equal(s.top_ids[-3:], f.top_ids)
    S = (V / 64 + 2 * math.log(V) + 96) * U
    assert (s.log_probs[-3:] - f.log_probs).abs().max() <= 2 * S + 8 * U * 20
    assert (D[-3:].float() - d.float()).abs().max() <= 2.0**-8


def test_repeats_streams_and_recorded_calls():
    announce("scores capture")
    logits, targets = problem((4,), 70000, "bf16", seed=9)
    x, t = logits.to(DEV).requires_grad_(), targets.to(DEV)

    def step():
        # (Nothing of autograd's graph is kept: it would hold x's node of an eager pass, whose stream is the default one, and a recorded
        # backward pass would hand its gradient over to that stream, which leaves the recording forked.)
        s = token_log_probs(x, t, entropy=True, top_k=8)
        (d,) = torch.autograd.grad(s.log_probs.sum() - s.entropy.sum(), x)
        return tuple(v.detach() for v in s) + (d,)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        with torch.no_grad():
            x.normal_()
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("R,V,k,dtype", [(5, 777, 3, lib.DTYPE_F32), (2, 70001, 20, lib.DTYPE_BF16), (1, 200000, 64, lib.DTYPE_F32)])
def test_entry_points_fill_every_byte_and_no_other(R, V, k, dtype):
    announce("scores entry", R, V, k, dtype)
    cabi = sequence_lib.load()
    es = 2 if dtype == lib.DTYPE_BF16 else 4
    logits, targets = problem((R,), V, "bf16" if es == 2 else "f32", seed=10)
    x, t = logits.to(DEV), targets.to(DEV)
    g = torch.randn((R,), device=DEV)
    sizes = dict(log_prob=R * 4, norm=R * 8, entropy=R * 4, top=R * k * 4, ids=R * k * 8, ws=cabi.rtn_token_log_probs_workspace_bytes(R, V, dtype, k), D=R * V * es)
    buf = {name: torch.full((n + 512,), 0xFF, dtype=torch.uint8, device=DEV) for name, n in sizes.items()}
    at = {name: b.data_ptr() + 256 for name, b in buf.items()}
    stream = torch.cuda.current_stream().cuda_stream
    assert cabi.rtn_token_log_probs_fwd(x.data_ptr(), 0, t.data_ptr(), R, V, dtype, k, at["log_prob"], at["norm"], at["entropy"], at["top"], at["ids"], at["ws"], sizes["ws"], stream) == 0
    assert cabi.rtn_token_log_probs_bwd(x.data_ptr(), 0, t.data_ptr(), at["norm"], at["entropy"], g.data_ptr(), None, at["D"], R, V, dtype, stream) == 0
    torch.cuda.synchronize()
    s = token_log_probs(x, t, entropy=True, top_k=k)

    def inside(name, ty):
        return buf[name][256 : 256 + sizes[name]].view(ty)

    assert torch.equal(inside("log_prob", torch.float32), s.log_probs) and torch.equal(inside("entropy", torch.float32), s.entropy)
    assert torch.equal(inside("ids", torch.int64).view(R, k), s.top_ids) and torch.equal(inside("top", torch.float32).view(R, k), s.top_log_probs)
    check(logits, targets, k, s, (g, None, inside("D", x.dtype).view(R, V)))
    for name, b in buf.items():
        assert bool((b[:256] == 0xFF).all()) and bool((b[256 + sizes[name] :] == 0xFF).all()), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [200, 1000, 5000])
def test_gradient_of_probabilities_that_are_no_normal_numbers(V, dtype):
    """
    A large error of the entropy makes normal numbers of them: p is below 2^-126, its products are not.

    (Bound: as above, and the entropy's own, 4 (1 + log V) S, times p and the entropy's error: the entropy is some 1e-32 here, and so is
    what the token with nearly all of the probability is made of.)
    """
    announce("scores small probabilities", V, dtype)
    logits = torch.linspace(-80.0, -103.0, V)[None].repeat(3, 1)
    logits[:, V // 3] = torch.tensor([0.0, 0.125, -0.25])
    logits = logits.to(_DTYPES[dtype])
    leaf, ge = logits.to(DEV).requires_grad_(), torch.tensor([1000.0, -300.0, 3.0], device=DEV)
    s = token_log_probs(leaf, None, entropy=True)
    (D,) = torch.autograd.grad(s.entropy, leaf, ge)
    check(logits, None, 0, s)
    _, entropy, _, _, log_p = ref.scores(array(logits))
    want = ref.scores_grad(array(logits), None, numpy.zeros(3), array(ge))
    S, h, made_of = (V / 64 + 2 * math.log(V) + 96) * U, entropy[:, None], numpy.exp(log_p) * numpy.abs(array(ge))[:, None]
    half = 2.0**-8 if dtype == "bf16" else U
    near(array(D), want, 4 * S * made_of * ((2 + numpy.abs(log_p) + h) * (numpy.abs(log_p) + h) + 1 + math.log(V)) + half * numpy.abs(want) + 2.0**-126)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(24, 1000), (300, 1000), (24, 1500), (24, 6000), (300, 6000), (24, 32000), (300, 32000), (24, 70001), (300, 70001)])
def test_first_logits_that_are_low(rows, V, dtype):
    """
    The largest logits far above those at the beginning of their row, by what a float32 sum of exponentials can just hold and by more; all of the
    later ones, or one in eight.  In rows of one wavefront, of several, and in pieces.

    (Sums relative to a logit up to 22 below the largest: an exponential of them is good to (22 + log V + 8 + 8) u, and what it takes to join
    the lanes', wavefronts' and pieces' sums is 23 additions, so that S as above has room for those and for half a unit each of the difference
    to the reference and of the logarithm, which are below 22 + log V: together V / 64 + 2 log V + 83.)
    """
    announce("scores low first logits", rows, V, dtype)
    logits, targets = problem((rows,), V, dtype, seed=V + rows, spread=1.0)
    where = torch.arange(V)
    for r in range(rows):
        low = (20.0, 60.0, 70.0, 76.0, 78.0, 80.0, 83.0, 85.0, 87.0, 88.0, 90.0, 130.0)[r % 12]
        lead = (512, 2048, 8192)[r // 12 % 3]
        high = where >= min(lead, V - 8)
        if r // 36 % 2:
            high &= where % 8 == 0
        logits[r][~high] -= low
        if r % 4 == 3:  # (all the high ones alike: the sums are as large as they get)
            logits[r][high] = 0.5
        if r % 3:
            targets[r] = V - 1 - int(high.flip(0).int().argmax())
    s, grads = run(logits, targets, 0)
    check(logits, targets, 0, s, grads)
    s, grads = run(logits, targets, 0, entropy=False)
    check(logits, targets, 0, s, grads)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(5, 1), (5, 3), (5, 7), (5, 8), (5, 9), (5, 12), (700, 12), (5, 64), (700, 64), (5, 90), (700, 200), (1100, 700), (1100, 2000), (5, 3000), (5, 40000)])
def test_alternatives_with_a_nan_anywhere(rows, V, dtype):
    """A NaN comes before everything, at the first index and the last as well, and NaN among themselves by index: every token is listed once."""
    announce("scores nan anywhere", rows, V, dtype)
    logits, _ = problem((rows,), V, dtype, seed=12)
    for r in range(rows):
        kind = r % 5
        if kind == 0:
            logits[r, 0] = float("nan")
        elif kind == 1:
            logits[r] = float("nan")
        elif kind == 2:
            logits[r, V - 1] = float("nan")
        elif kind == 3:
            logits[r, 0] = logits[r, V // 2] = float("nan")
            logits[r, V // 3] = -INF
        else:
            logits[r, V // 2] = INF
    for k in sorted({1, min(V, 8), min(V, 9), min(V, 64)}):
        s = token_log_probs(logits.to(DEV), top_k=k)
        with numpy.errstate(invalid="ignore"):
            _, _, _, ids, _ = ref.scores(array(logits), None, k)
        assert numpy.array_equal(s.top_ids.cpu().numpy(), ids), k
