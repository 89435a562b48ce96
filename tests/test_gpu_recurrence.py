"""
The gated linear recurrence and its gradient on the GPU against their definitions in 64 bits.

Error bounds: a frame adds to the state's error at most 32 u times the largest magnitude M that a state has (u = 2^-24: gates to
about 4 u of themselves or 8 u absolute, two products, one sum), and a frame's error reaches later ones times their forget gates; N
is the largest sum of such products in the problem.  Twice that for sums in another order: 64 u N M.  The gradient's sums have
the same form in the errors' magnitude G, and a factor 1 + M from the states they are multiplied with.  bfloat16 results: half a unit in the
last place more, 2^-8 of the value.
"""

from __future__ import annotations

import numpy
import pytest
import torch

import _sequence_ref as ref
from _gpu_util import announce
from returnn_amd import lib, sequence_lib
from returnn_amd.recurrence import GatedRecurrence, gated_recurrence

pytestmark = pytest.mark.gpu
U = 2.0**-24
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda:0"


def problem(T, B, n, dtype, lens=None, seed=0, keep=2.0):
    rng = numpy.random.default_rng(seed)
    x = rng.normal(size=(T, B, 4 * n)).astype(numpy.float32)
    x[..., 2 * n : 3 * n] += keep
    x = torch.from_numpy(x).to(_DTYPES[dtype])
    c0 = torch.from_numpy(rng.normal(size=(B, n)).astype(numpy.float32))
    dy = torch.from_numpy(rng.normal(size=(T, B, n)).astype(numpy.float32)).to(_DTYPES[dtype])
    dc = torch.from_numpy(rng.normal(size=(B, n)).astype(numpy.float32))
    if lens == "ragged":
        lens = rng.integers(0, T + 1, size=(B,))
        lens[0] = T
        if B > 1:
            lens[1] = 0
    return x, c0, dy, dc, lens


def array(t):
    return t.detach().double().cpu().numpy()


def check_forward(y, c, x, c0, lens, direction):
    want_y, want_c, info = ref.recurrence(array(x), None if c0 is None else array(c0), lens, direction)
    bound = 64 * U * info["most"] * info["largest"]
    half = 2.0**-8 if y.dtype == torch.bfloat16 else U
    assert numpy.all(numpy.abs(array(y) - want_y) <= bound + half * numpy.abs(want_y)), numpy.abs(array(y) - want_y).max() / bound
    assert numpy.all(numpy.abs(array(c) - want_c) <= bound), numpy.abs(array(c) - want_c).max() / bound


def check_gradient(dx, dc0, x, dy, dc, c0, lens, direction):
    want_dx, want_dc0, G, most_g = ref.recurrence_grad(array(x), array(dy), array(dc), None if c0 is None else array(c0), lens, direction)
    _, _, info = ref.recurrence(array(x), None if c0 is None else array(c0), lens, direction)
    G = max(G, numpy.abs(array(dy)).max(initial=0.0))
    bound = 64 * U * max(info["most"], most_g) * G * (1 + info["largest"])
    half = 2.0**-8 if dx.dtype == torch.bfloat16 else U
    assert numpy.all(numpy.abs(array(dx) - want_dx) <= bound + half * numpy.abs(want_dx)), numpy.abs(array(dx) - want_dx).max() / bound
    if dc0 is not None:
        assert numpy.all(numpy.abs(array(dc0) - want_dc0) <= bound), numpy.abs(array(dc0) - want_dc0).max() / bound


def run(x, c0, dy, dc, lens, direction, train):
    xd = x.to(DEV).requires_grad_(train)
    cd = None if c0 is None else c0.to(DEV).requires_grad_(train)
    ld = None if lens is None else torch.as_tensor(lens).to(DEV)
    y, c = gated_recurrence(xd, state=cd, seq_lens=ld, direction=direction)
    if not train:
        return y, c
    grads = torch.autograd.grad((y, c), (xd,) if cd is None else (xd, cd), (dy.to(DEV), dc.to(DEV)))
    return (y, c) + tuple(grads) + ((None,) if cd is None else ())


SHAPES = [
    (1, 1, 1), (1, 12, 64), (2, 3, 5), (15, 2, 63), (16, 2, 64), (17, 2, 65), (31, 4, 127), (33, 1, 128), (64, 3, 129), (100, 5, 200), (127, 1, 130), (129, 2, 96),
    (257, 3, 31), (300, 70, 8), (513, 1, 260), (1000, 2, 64), (1025, 1, 2), (2049, 3, 33), (5000, 1, 66),
]  # fmt: skip


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,B,n", SHAPES)
def test_against_the_definition(T, B, n, dtype):
    for direction, lens in ((1, None), (-1, "ragged"), (1, "ragged"), (-1, None)):
        announce("recurrence", T, B, n, dtype, direction, lens)
        x, c0, dy, dc, lens = problem(T, B, n, dtype, lens, seed=T + B + n)
        y, c = run(x, c0, dy, dc, lens, direction, False)
        check_forward(y, c, x, c0, lens, direction)
        y2, c2, dx, dc0 = run(x, c0, dy, dc, lens, direction, True)
        assert torch.equal(y, y2) and torch.equal(c, c2)
        check_gradient(dx, dc0, x, dy, dc, c0, lens, direction)


@pytest.mark.parametrize("T,B,n,dtype", [(131, 70, 201, "f32"), (70, 230, 201, "f32"), (131, 140, 201, "bf16"), (67, 460, 130, "bf16"), (90, 48, 640, "f32"), (80, 64, 512, "bf16")])
def test_many_rows(T, B, n, dtype):
    """Enough of them for lanes that have more channels, in one round and in several; and rows with a pitch."""
    announce("recurrence many rows", T, B, n, dtype)
    for direction in (1, -1):
        x, c0, dy, dc, lens = problem(T, B, n, dtype, "ragged", seed=T + B)
        y, c, dx, dc0 = run(x, c0, dy, dc, lens, direction, True)
        check_forward(y, c, x, c0, lens, direction)
        check_gradient(dx, dc0, x, dy, dc, c0, lens, direction)
        wide = torch.full((T, B, 4 * n + 3), float("nan"), dtype=x.dtype, device=DEV)
        wide[..., 1 : 4 * n + 1] = x.to(DEV)
        y2, c2 = gated_recurrence(wide[..., 1 : 4 * n + 1], state=c0.to(DEV), seq_lens=torch.as_tensor(lens), direction=direction)
        assert torch.equal(y, y2) and torch.equal(c, c2)


@pytest.mark.parametrize("keep", [-30.0, 0.0, 8.0, 100.0])
def test_gates_that_forget_or_keep_everything(keep):
    """Products of many forget gates that underflow, and states that add up over all frames."""
    announce("recurrence keep", keep)
    for dtype in ("f32", "bf16"):
        x, c0, dy, dc, lens = problem(700, 2, 70, dtype, "ragged", seed=5, keep=keep)
        y, c, dx, dc0 = run(x, c0, dy, dc, lens, 1, True)
        check_forward(y, c, x, c0, lens, 1)
        check_gradient(dx, dc0, x, dy, dc, c0, lens, 1)


def test_saturated_gates_are_finite():
    """Gates far outside the range of the exponential, both ways."""
    for dtype in ("f32", "bf16"):
        announce("recurrence saturated", dtype)
        x, c0, dy, dc, _ = problem(40, 2, 64, dtype, seed=6)
        x = (x.float() * 1e4).to(x.dtype)
        y, c, dx, dc0 = run(x, c0, dy, dc, None, 1, True)
        check_forward(y, c, x, c0, None, 1)
        check_gradient(dx, dc0, x, dy, dc, c0, None, 1)


@pytest.mark.parametrize("direction", [1, -1])
@pytest.mark.parametrize("T,n", [(40, 64), (300, 65), (1100, 128)])
def test_frames_past_the_end_are_not_read(T, n, direction):
    """NaN in the padding of input and error stays there; lengths beyond the range are cut."""
    for dtype in ("f32", "bf16"):
        announce("recurrence padding", T, n, dtype, direction)
        x, c0, dy, dc, _ = problem(T, 5, n, dtype, seed=7)
        lens = numpy.array([T, 0, T // 2, 1, T - 1])
        for b, l in enumerate(lens):
            x[l:, b] = float("nan")
            dy[l:, b] = float("nan")
        y, c, dx, dc0 = run(x, c0, dy, dc, numpy.array([T + 7, -3, T // 2, 1, T - 1]), direction, True)
        dy0 = torch.nan_to_num(dy.float()).to(dy.dtype)
        check_forward(y, c, x, c0, lens, direction)
        check_gradient(dx, dc0, x, dy0, dc, c0, lens, direction)
        assert torch.equal(c[1], c0[1].to(DEV)) and torch.equal(dc0[1], dc[1].to(DEV))


def test_a_nan_stays_in_its_sequence_and_channel():
    announce("recurrence nan")
    x, c0, dy, dc, _ = problem(300, 3, 66, "f32", seed=8)
    clean, _ = run(x, c0, dy, dc, None, 1, False)
    x[150, 1, 2 * 66 + 10] = float("nan")
    y, c = run(x, c0, dy, dc, None, 1, False)
    hit = torch.isnan(y)
    want = torch.zeros_like(hit)
    want[150:, 1, 10] = True
    assert torch.equal(hit, want) and torch.isnan(c[1, 10]) and int(torch.isnan(c).sum()) == 1
    assert torch.equal(y[~hit], clean[~hit])


def test_gradient_against_differences():
    """Of the definition's values, not of its gradient's formula."""
    announce("recurrence differences")
    T, B, n, h = 21, 2, 3, 1e-5
    x, c0, dy, dc, _ = problem(T, B, n, "f32", seed=9)
    lens = numpy.array([T, 13])
    _, _, dx, dc0 = run(x, c0, dy, dc, lens, -1, True)
    xa, ca = array(x), array(c0)

    def value():
        y, c, _ = ref.recurrence(xa, ca, lens, -1)
        return (y * array(dy)).sum() + (c * array(dc)).sum()

    for a, d in ((xa, dx), (ca, dc0)):
        for at in list(numpy.ndindex(a.shape))[::5]:
            old = a[at]
            a[at] = old + h
            up = value()
            a[at] = old - h
            down = value()
            a[at] = old
            # (differences to 1e-8; the gradient to 64 u N G (1 + M) with N, G and M below 10)
            assert abs((up - down) / (2 * h) - float(d[at])) < 64 * U * 1000


@pytest.mark.parametrize("T,B,n,dtype", [(70, 3, 64, "bf16"), (70, 3, 64, "f32"), (9, 2, 33, "bf16"), (300, 2, 130, "f32")])
def test_strides_and_orders(T, B, n, dtype):
    """Slices of a wider projection, rows at odd addresses, transposed and expanded tensors."""
    announce("recurrence strides", T, B, n, dtype)
    x, c0, dy, dc, lens = problem(T, B, n, dtype, "ragged", seed=10)
    want = run(x, c0, dy, dc, lens, 1, True)
    wide = torch.full((T, B, 4 * n + 37), float("nan"), dtype=x.dtype, device=DEV)
    wide_dy = torch.full((T, B, 2 * n + 3), float("nan"), dtype=x.dtype, device=DEV)
    for at in (0, 1, 8, 37):
        xs, ds = wide[..., at : at + 4 * n], wide_dy[..., at % 4 : at % 4 + n]
        xs.copy_(x)
        ds.copy_(dy)
        leaf = xs.detach().requires_grad_()
        cd = c0.to(DEV).requires_grad_()
        y, c = gated_recurrence(leaf, state=cd, seq_lens=torch.as_tensor(lens), direction=1)
        got = (y, c) + torch.autograd.grad((y, c), (leaf, cd), (ds, dc.to(DEV)))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    batch_major = x.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    y, _ = gated_recurrence(batch_major, state=c0.to(DEV), seq_lens=torch.as_tensor(lens), direction=1)
    assert torch.equal(y, want[0])
    one = x[:, :1].to(DEV).expand(T, 4, 4 * n)
    y, c = gated_recurrence(one)
    assert torch.equal(y[:, 0], y[:, 3]) and torch.equal(c[0], c[3])
    # the error of a sum: one number, expanded
    leaf = x.to(DEV).requires_grad_()
    y, _ = gated_recurrence(leaf)
    (dx,) = torch.autograd.grad(y.sum(), leaf)
    check_gradient(dx, None, x, torch.ones_like(dy), torch.zeros_like(dc), None, None, 1)


def test_parts_of_the_gradient():
    """Only the output or only the state used; no state given; lengths of other types."""
    announce("recurrence parts")
    T, B, n = 150, 3, 40
    x, c0, dy, dc, lens = problem(T, B, n, "f32", "ragged", seed=11)
    xd = x.to(DEV).requires_grad_()
    y, c = gated_recurrence(xd, seq_lens=torch.as_tensor(lens, dtype=torch.int32))
    check_forward(y, c, x, None, lens, 1)
    (dx,) = torch.autograd.grad(y, xd, dy.to(DEV), retain_graph=True)
    check_gradient(dx, None, x, dy, torch.zeros_like(dc), None, lens, 1)
    (dx,) = torch.autograd.grad(c, xd, dc.to(DEV))
    check_gradient(dx, None, x, torch.zeros_like(dy), dc, None, lens, 1)
    half = c0.to(DEV).bfloat16().requires_grad_()
    y, c = gated_recurrence(x.to(DEV), state=half)
    (d,) = torch.autograd.grad(c.sum(), half)
    assert d.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="gradient"):
        y, _ = gated_recurrence(xd)
        torch.autograd.grad(y.sum(), xd, create_graph=True)


def test_one_step_is_a_sequence_of_one_frame():
    announce("recurrence step")
    for dtype, B, n in (("bf16", 12, 1024), ("f32", 3, 33), ("bf16", 1, 7)):
        x, c0, _, _, _ = problem(30, B, n, dtype, seed=12)
        y, c = gated_recurrence(x.to(DEV), state=c0.to(DEV))
        s = c0.to(DEV)
        for t in range(30):
            step, s = gated_recurrence(x[t].to(DEV), state=s)
            bound = 64 * U * 30 * 40
            assert torch.all((step.float() - y[t].float()).abs() <= bound + 2.0**-8 * y[t].float().abs() * (dtype == "bf16"))
        assert torch.all((s - c).abs() <= bound)


def test_empty():
    announce("recurrence empty")
    for T, B, n in ((0, 3, 8), (5, 0, 8), (5, 3, 0)):
        x = torch.zeros((T, B, 4 * n), device=DEV, requires_grad=True)
        c0 = torch.randn((B, n), device=DEV).requires_grad_()
        y, c = gated_recurrence(x, state=c0)
        assert y.shape == (T, B, n) and torch.equal(c, c0)
        dx, dc0 = torch.autograd.grad((y, c), (x, c0), (torch.ones_like(y), torch.ones_like(c)))
        assert dx.shape == x.shape and torch.equal(dc0, torch.ones_like(c0))


def test_refusals():
    announce("recurrence refusals")
    x = torch.zeros((4, 3, 32), device=DEV)
    for bad in (dict(state=torch.zeros((3, 7), device=DEV)), dict(state=torch.zeros((3, 8))), dict(seq_lens=torch.zeros((4,), dtype=torch.int64)),
                dict(seq_lens=torch.zeros((3,))), dict(direction=0), dict(state=torch.zeros((3, 8), dtype=torch.int64, device=DEV))):  # fmt: skip
        with pytest.raises(RuntimeError):
            gated_recurrence(x, **bad)
    for t in (x[..., :30], x[0, 0], x.half(), x.double(), x.long()):
        with pytest.raises(RuntimeError):
            gated_recurrence(t)
    torch.cuda.synchronize()


def test_beyond_32_bits():
    """More than 2^32 bytes and 2^31 elements of gates; the last sequence against the definition."""
    announce("recurrence beyond 32 bits")
    T, B, n = 530, 256, 4096
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty((T, B, 4 * n), dtype=torch.bfloat16, device=DEV).normal_(generator=gen).requires_grad_()
    y, c = gated_recurrence(x)
    dy = torch.empty_like(y).normal_(generator=gen)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert x.numel() > 2**31
    few = x.detach()[:, -1:]
    check_forward(y[:, -1:], c[-1:], few, None, None, 1)
    check_gradient(dx[:, -1:], None, few, dy[:, -1:], torch.zeros((1, n)), None, None, 1)


def test_other_stream_and_repeats_are_bit_for_bit():
    announce("recurrence streams")
    x, c0, dy, dc, lens = problem(3000, 2, 130, "bf16", "ragged", seed=13)
    want = run(x, c0, dy, dc, lens, 1, True)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(stream):
            got = run(x, c0, dy, dc, lens, 1, True)
        stream.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_recorded_calls():
    """Forward and gradient in a graph, replayed with eager work in between; every replay against the eager result."""
    announce("recurrence capture")
    T, B, n = 700, 3, 130
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((T, B, 4 * n), device=DEV, generator=gen).requires_grad_()
    c0 = torch.randn((B, n), device=DEV, generator=gen).requires_grad_()
    lens = torch.tensor([T, 333, 0], device=DEV)
    dy = torch.randn((T, B, n), device=DEV, generator=gen)

    def step():
        y, c = gated_recurrence(x, state=c0, seq_lens=lens)
        return (y.detach(), c.detach()) + torch.autograd.grad((y, c), (x, c0), (dy, torch.ones_like(c)))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.normal_(generator=gen)
            c0.normal_(generator=gen)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


def test_layer_trains():
    """The layer's parameters against autograd's gradient of the definition in float64 on the CPU."""
    announce("recurrence layer")
    torch.manual_seed(0)
    T, B, i, n = 12, 3, 6, 5
    m = GatedRecurrence(i, n, device=DEV)
    x = torch.randn((T, B, i), device=DEV)
    y, _ = m(x, seq_lens=torch.tensor([12, 5, 9]))
    y.square().sum().backward()
    ff, bias = m.ff.detach().double().cpu().requires_grad_(), m.bias.detach().double().cpu().requires_grad_()
    gates = torch.nn.functional.linear(x.double().cpu(), ff, bias)
    c, loss = torch.zeros((B, n), dtype=torch.float64), 0.0
    for t in range(T):
        inside = (t < torch.tensor([12, 5, 9]))[:, None]
        z, a, f, o = gates[t].chunk(4, dim=-1)
        c = torch.where(inside, torch.sigmoid(f) * c + torch.sigmoid(a) * torch.tanh(z), c)
        loss = loss + torch.where(inside, torch.sigmoid(o) * c, 0.0).square().sum()
    loss.backward()
    # (float32 products of some ten terms, sums over T B = 36 rows: 1e-5 of the largest is hundreds of u)
    for got, want in ((m.ff.grad, ff.grad), (m.bias.grad, bias.grad)):
        assert (got.double().cpu() - want).abs().max() <= 1e-5 * want.abs().max()


def test_entry_points_fill_every_byte_and_no_other():
    """Through the C entries, into buffers of NaN with guards around them."""
    announce("recurrence entry")
    cabi = sequence_lib.load()
    T, B, n = 213, 3, 70
    x, c0, dy, dc, lens = problem(T, B, n, "bf16", "ragged", seed=14)
    want = run(x, c0, dy, dc, lens, -1, True)
    xd, cd, dyd, dcd, ld = x.to(DEV), c0.to(DEV), dy.to(DEV), dc.to(DEV), torch.as_tensor(lens).to(DEV)

    def guarded(nbytes):
        return torch.full((nbytes + 512,), 0xFF, dtype=torch.uint8, device=DEV)

    sizes = dict(y=T * B * n * 2, c=B * n * 4, dx=T * B * 4 * n * 2, dc0=B * n * 4, saved=cabi.rtn_gated_recurrence_saved_bytes(T, B, n, lib.DTYPE_BF16),
                 fwd=cabi.rtn_gated_recurrence_fwd_workspace_bytes(T, B, n, lib.DTYPE_BF16), bwd=cabi.rtn_gated_recurrence_bwd_workspace_bytes(T, B, n, lib.DTYPE_BF16))  # fmt: skip
    buf = {k: guarded(v) for k, v in sizes.items()}
    at = {k: v.data_ptr() + 256 for k, v in buf.items()}
    stream = torch.cuda.current_stream().cuda_stream
    assert cabi.rtn_gated_recurrence_fwd(xd.data_ptr(), 0, cd.data_ptr(), ld.data_ptr(), at["y"], at["c"], at["saved"], T, B, n, lib.DTYPE_BF16, -1, at["fwd"], sizes["fwd"], stream) == 0
    assert cabi.rtn_gated_recurrence_bwd(xd.data_ptr(), 0, cd.data_ptr(), ld.data_ptr(), at["saved"], dyd.data_ptr(), 0, dcd.data_ptr(), at["dx"], at["dc0"], T, B, n,
                                         lib.DTYPE_BF16, -1, at["bwd"], sizes["bwd"], stream) == 0  # fmt: skip
    torch.cuda.synchronize()
    for key, t in zip(("y", "c", "dx", "dc0"), want):
        got = buf[key][256 : 256 + sizes[key]].view(t.dtype).view(t.shape)
        assert torch.equal(got, t.detach()), key
    for key, b in buf.items():
        assert bool((b[:256] == 0xFF).all()) and bool((b[256 + sizes[key] :] == 0xFF).all()), key


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,B,n", [(1, 3, 64), (6, 2, 33), (40, 3, 130), (70, 64, 512), (300, 2, 96)])
def test_small_cell_inputs(T, B, n, dtype):
    """
    Cell inputs down to 1e-30 and no state: everything is as small as they are, and good to as much of itself.

    (All terms have one sign.  The cell input's function is good to 2^-15 of itself in bfloat16, to 4 u in float32; a state whose products of forget gates
    have up to T factors, and its gradient, to (T + 8) 2^-22 more with the roundings of sums and products in any order; bfloat16 results to 2^-8 more.)
    """
    announce("recurrence small cell inputs", T, B, n, dtype)
    x, _, dy, dc, _ = problem(T, B, n, dtype, seed=16)
    size = torch.logspace(0, -30, n) * torch.linspace(0.5, 1.0, T * B).view(T, B, 1)
    x[..., :n] = size.to(x.dtype)
    dy, dc = dy.abs(), dc.abs()
    y, c, dx, _ = run(x, torch.zeros((B, n)), dy, dc, None, 1, True)
    want_y, want_c, _ = ref.recurrence(array(x))
    want_dx, _, _, _ = ref.recurrence_grad(array(x), array(dy), array(dc))
    rel = (2.0**-15 if dtype == "bf16" else 0.0) + (T + 8) * 2.0**-22
    half = 2.0**-8 if dtype == "bf16" else 0.0
    assert numpy.all(numpy.abs(array(c) - want_c) <= rel * want_c)
    assert numpy.all(numpy.abs(array(y) - want_y) <= (rel + half) * want_y)
    # (the input gate's error is proportional to the cell input; of the sigmoid's slope, i (1 - i), 1 - i is good to 4 u of 1, here 1 - i > 0.005)
    d, want = array(dx)[..., n : 2 * n], want_dx[..., n : 2 * n]
    assert numpy.all(numpy.abs(d - want) <= (2 * rel + half + 800 * U) * numpy.abs(want) + 2.0**-126)
