"""
CPU-side checks of the sequence operators: the library loads and exports what its header declares, refusals come before
any launch, the definitions that the GPU tests compare with hold (published vectors, differences, closed forms).
"""

from __future__ import annotations

import os
import re
import subprocess

import numpy
import pytest
import torch

import _sequence_ref as ref
import test_generated_code as generated
from returnn_amd import build, lib, sequence_lib
from returnn_amd.dropout import Dropout, dropout
from returnn_amd.language_model import RecurrentLanguageModel
from returnn_amd.recurrence import GatedRecurrence, gated_recurrence
from returnn_amd.scoring import token_log_probs

_root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16 = lib.DTYPE_F32, lib.DTYPE_BF16


@pytest.fixture(scope="module")
def cabi():
    if not os.path.exists(build.SEQUENCE_LIB_PATH):
        build.build_library()
    return sequence_lib.load()


def test_header_symbols_are_exported(cabi):
    header = open(os.path.join(_root, "include", "rtn_sequence_ops.h")).read()
    declared = set(re.findall(r"^(?:int|size_t|const char\*) (rtn_[a-z0-9_]+)\(", header, re.M))
    assert declared == set(sequence_lib.SYMBOLS)
    for name in declared:
        assert getattr(cabi, name) is not None
    assert re.findall(r"ABI version of this header: (\d+)\.", header) == [str(sequence_lib.EXPECTED_ABI)]
    assert cabi.rtn_sequence_ops_abi_version() == sequence_lib.EXPECTED_ABI


def test_loader_refuses_another_abi_version(monkeypatch):
    monkeypatch.setattr(sequence_lib, "_lib", None)
    monkeypatch.setattr(sequence_lib, "EXPECTED_ABI", sequence_lib.EXPECTED_ABI + 1)
    with pytest.raises(lib.NativeLibraryMismatch):
        sequence_lib.load()


def test_the_library_is_never_built_silently(monkeypatch, tmp_path):
    monkeypatch.setattr(sequence_lib, "_lib", None)
    monkeypatch.setattr(build, "SEQUENCE_LIB_PATH", str(tmp_path / "none.so"))
    with pytest.raises(lib.NativeLibraryMissing):
        sequence_lib.load()


P = 1 << 20  # an address that is never looked at: every call below is refused by the host, or has nothing to do


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(T=-1), lib.RTN_ERR_SHAPE), (dict(B=-1), lib.RTN_ERR_SHAPE), (dict(n=-2), lib.RTN_ERR_SHAPE), (dict(ldX=31), lib.RTN_ERR_SHAPE),
        (dict(dtype=2), lib.RTN_ERR_ARG), (dict(direction=0), lib.RTN_ERR_RANGE), (dict(direction=2), lib.RTN_ERR_RANGE),
        (dict(X=None), lib.RTN_ERR_ARG), (dict(Y=None), lib.RTN_ERR_ARG), (dict(cN=None), lib.RTN_ERR_ARG),
        (dict(X=P + 1), lib.RTN_ERR_ARG), (dict(X=P + 2, dtype=F32), lib.RTN_ERR_ARG), (dict(c0=P + 2), lib.RTN_ERR_ARG), (dict(lens=P + 4), lib.RTN_ERR_ARG),
        (dict(Y=P + 1), lib.RTN_ERR_ARG), (dict(cN=P + 1), lib.RTN_ERR_ARG), (dict(saved=P + 4), lib.RTN_ERR_ARG),
        (dict(B=0), lib.RTN_OK), (dict(n=0), lib.RTN_OK),
    ],
)  # fmt: skip
def test_recurrence_refusals(cabi, change, code):
    a = dict(X=P, ldX=0, c0=P, lens=P, Y=P, cN=P, saved=P, T=5, B=3, n=8, dtype=BF16, direction=1)
    a.update(change)
    assert cabi.rtn_gated_recurrence_fwd(*a.values(), None, 0, None) == code
    assert bool(sequence_lib.last_error()) == (code != lib.RTN_OK)


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(T=-1), lib.RTN_ERR_SHAPE), (dict(ldX=31), lib.RTN_ERR_SHAPE), (dict(ldDY=7), lib.RTN_ERR_SHAPE), (dict(dtype=5), lib.RTN_ERR_ARG),
        (dict(direction=0), lib.RTN_ERR_RANGE), (dict(saved=None), lib.RTN_ERR_ARG), (dict(DY=None), lib.RTN_ERR_ARG), (dict(DX=None), lib.RTN_ERR_ARG),
        (dict(Dc0=None), lib.RTN_ERR_ARG), (dict(DY=P + 1), lib.RTN_ERR_ARG), (dict(DX=P + 1), lib.RTN_ERR_ARG), (dict(DcN=P + 2), lib.RTN_ERR_ARG),
        (dict(B=0), lib.RTN_OK),
    ],
)  # fmt: skip
def test_recurrence_gradient_refusals(cabi, change, code):
    a = dict(X=P, ldX=0, c0=P, lens=P, saved=P, DY=P, ldDY=0, DcN=P, DX=P, Dc0=P, T=5, B=3, n=8, dtype=BF16, direction=1)
    a.update(change)
    assert cabi.rtn_gated_recurrence_bwd(*a.values(), None, 0, None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(times=-1), lib.RTN_ERR_SHAPE), (dict(rows=-1), lib.RTN_ERR_SHAPE), (dict(width=-1), lib.RTN_ERR_SHAPE), (dict(ldx=7), lib.RTN_ERR_SHAPE),
        (dict(ldr=7), lib.RTN_ERR_SHAPE), (dict(dtype=-1), lib.RTN_ERR_ARG), (dict(threshold=-1), lib.RTN_ERR_RANGE), (dict(threshold=65537), lib.RTN_ERR_RANGE),
        (dict(x=None), lib.RTN_ERR_ARG), (dict(y=None), lib.RTN_ERR_ARG), (dict(x=P + 1), lib.RTN_ERR_ARG), (dict(residual=P + 1), lib.RTN_ERR_ARG),
        (dict(offset_ptr=P + 4), lib.RTN_ERR_ARG), (dict(rows=0), lib.RTN_OK), (dict(width=0), lib.RTN_OK), (dict(times=0), lib.RTN_OK),
    ],
)  # fmt: skip
def test_dropout_refusals(cabi, change, code):
    a = dict(x=P, ldx=0, residual=P, ldr=0, y=P, times=3, rows=4, width=8, dtype=BF16, threshold=100, seed=1, offset=2, offset_ptr=None, same=0)
    a.update(change)
    assert cabi.rtn_dropout(*a.values(), None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(rows=-1), lib.RTN_ERR_SHAPE), (dict(V=-1), lib.RTN_ERR_SHAPE), (dict(V=0, top_k=0), lib.RTN_ERR_SHAPE), (dict(V=1 << 31), lib.RTN_ERR_SHAPE),
        (dict(rows=1 << 31), lib.RTN_ERR_SHAPE), (dict(ld=99), lib.RTN_ERR_SHAPE), (dict(dtype=3), lib.RTN_ERR_ARG), (dict(top_k=-1), lib.RTN_ERR_RANGE),
        (dict(top_k=65), lib.RTN_ERR_RANGE), (dict(top_k=5, V=4), lib.RTN_ERR_RANGE), (dict(logits=None), lib.RTN_ERR_ARG), (dict(targets=None), lib.RTN_ERR_ARG),
        (dict(top_ids=None), lib.RTN_ERR_ARG), (dict(top=None), lib.RTN_ERR_ARG), (dict(logits=P + 1), lib.RTN_ERR_ARG), (dict(targets=P + 4), lib.RTN_ERR_ARG),
        (dict(log_prob=P + 2), lib.RTN_ERR_ARG), (dict(norm=P + 4), lib.RTN_ERR_ARG), (dict(top_ids=P + 4), lib.RTN_ERR_ARG), (dict(rows=0), lib.RTN_OK),
    ],
)  # fmt: skip
def test_scores_refusals(cabi, change, code):
    a = dict(logits=P, ld=0, targets=P, rows=6, V=100, dtype=BF16, top_k=4, log_prob=P, norm=P, entropy=P, top=P, top_ids=P)
    a.update(change)
    assert cabi.rtn_token_log_probs_fwd(*a.values(), None, 0, None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(rows=-1), lib.RTN_ERR_SHAPE), (dict(ld=99), lib.RTN_ERR_SHAPE), (dict(norm=None), lib.RTN_ERR_ARG), (dict(D=None), lib.RTN_ERR_ARG),
        (dict(entropy=None), lib.RTN_ERR_ARG), (dict(targets=None), lib.RTN_ERR_ARG), (dict(D=P + 1), lib.RTN_ERR_ARG), (dict(rows=0), lib.RTN_OK),
    ],
)  # fmt: skip
def test_scores_gradient_refusals(cabi, change, code):
    a = dict(logits=P, ld=0, targets=P, norm=P, entropy=P, d_log_prob=P, d_entropy=P, D=P, rows=6, V=100, dtype=BF16)
    a.update(change)
    assert cabi.rtn_token_log_probs_bwd(*a.values(), None) == code


def test_cpu_tensors_and_bad_arguments_are_refused(cabi):
    x = torch.zeros((2, 3, 8))
    with pytest.raises(RuntimeError, match="HIP"):
        gated_recurrence(x)
    with pytest.raises(RuntimeError, match="HIP"):
        GatedRecurrence(5, 2)(torch.zeros((2, 3, 5)))
    with pytest.raises(RuntimeError, match="HIP"):
        dropout(x, 0.5, seed=1)
    with pytest.raises(RuntimeError, match="HIP"):
        token_log_probs(x)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            dropout(x, p, seed=1)
        with pytest.raises(ValueError):
            Dropout(p)
    with pytest.raises(ValueError):
        GatedRecurrence(5, 2)(torch.zeros((2, 3, 4)))


def test_dropout_module_in_evaluation_is_the_identity():
    x, r = torch.randn((3, 4)), torch.randn((3, 4))
    m = Dropout(0.5).eval()
    assert m(x) is x and torch.equal(m(x, residual=r), x + r) and m.offset == 0


# ---- the definitions that the GPU tests compare with ----
@pytest.mark.parametrize(
    "counter,key,want",
    [  # the published vectors of the generator
        ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
        ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
        ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
    ],
)
def test_philox_vectors(counter, key, want):
    assert tuple(ref.philox(counter, key)) == want


def test_draws_are_even():
    """Of 64 Ki draws the share below a threshold is that of the threshold, within five standard deviations."""
    d = ref.draws(0, 1 << 16, 12345, 7)
    for p in (0.1, 0.5, 0.9):
        assert abs((d < p * 65536).mean() - p) < 5 * numpy.sqrt(p * (1 - p) / len(d))


@pytest.mark.parametrize("direction", [1, -1])
def test_recurrence_gradient_against_differences(direction):
    rng = numpy.random.default_rng(3)
    T, B, n = 7, 3, 2
    x, c0, lens = rng.normal(size=(T, B, 4 * n)), rng.normal(size=(B, n)), [7, 0, 4]
    dy, dc = rng.normal(size=(T, B, n)), rng.normal(size=(B, n))
    dx, dc0, _, _ = ref.recurrence_grad(x, dy, dc, c0, lens, direction)

    def value(x, c0):
        y, c, _ = ref.recurrence(x, c0, lens, direction)
        return (y * dy).sum() + (c * dc).sum()

    h = 1e-5  # (errors of h^2 and 1e-16 / h)
    for a, d in ((x, dx), (c0, dc0)):
        for at in numpy.ndindex(a.shape):
            old = a[at]
            a[at] = old + h
            up = value(x, c0)
            a[at] = old - h
            down = value(x, c0)
            a[at] = old
            assert abs((up - down) / (2 * h) - d[at]) < 1e-8


def test_scores_gradient_against_differences():
    rng = numpy.random.default_rng(4)
    R, V = 4, 9
    x, targets = rng.normal(size=(R, V)), numpy.array([3, -1, 8, 0])
    g, ge = rng.normal(size=R), rng.normal(size=R)
    d = ref.scores_grad(x, targets, g, ge)

    def value():
        lp, h, _, _, _ = ref.scores(x, targets)
        return (lp * g).sum() + (h * ge).sum()

    h = 1e-5
    for at in numpy.ndindex(x.shape):
        old = x[at]
        x[at] = old + h
        up = value()
        x[at] = old - h
        down = value()
        x[at] = old
        assert abs((up - down) / (2 * h) - d[at]) < 1e-8


def test_no_kernel_loses_a_copy(tmp_path):
    """As for the LSTM kernels: no value is copied between the end of a masked block and the switch back to all lanes."""
    if not os.path.exists(build.SEQUENCE_LIB_PATH) or not os.path.exists(generated.OBJDUMP):
        pytest.skip("no library or no llvm-objdump")
    with open(build.SEQUENCE_LIB_PATH, "rb") as f:
        objects = list(generated._code_objects(f.read()))
    assert len(objects) == 1
    path = tmp_path / "code.elf"
    path.write_bytes(objects[0])
    lines = subprocess.run([generated.OBJDUMP, "-d", str(path)], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines(keepends=True)
    assert sum("k_recurrence" in line for line in lines if line.endswith(">:\n")) > 0
    assert not generated.lost_copies(lines)


def test_launches_of_more_threads_than_32_bits_count_are_refused(cabi):
    """Sizes that the types of the arguments can hold, but a launch cannot: refused as a shape, before anything is enqueued."""
    for T, B, n, dtype in ((5, (1 << 31) - 1, 8, BF16), (100, 1 << 24, 64, F32)):
        assert cabi.rtn_gated_recurrence_fwd(P, 0, P, P, P, P, P, T, B, n, dtype, 1, None, 0, None) == lib.RTN_ERR_SHAPE
        assert cabi.rtn_gated_recurrence_bwd(P, 0, P, P, P, P, 0, P, P, P, T, B, n, dtype, 1, None, 0, None) == lib.RTN_ERR_SHAPE
    for width, ldx in ((8, 0), (8, 16)):
        assert cabi.rtn_dropout(P, ldx, None, 0, P, 1, 1 << 37, width, BF16, 100, 1, 2, None, 0, None) == lib.RTN_ERR_SHAPE
    for rows, V, top_k in ((1 << 30, 8, 1), (1 << 27, 300, 9), (1 << 23, 20000, 1), (1 << 28, 1000, 0), (1 << 25, 6000, 0)):
        assert cabi.rtn_token_log_probs_fwd(P, 0, P, rows, V, BF16, top_k, P, P, P, P, P, None, 0, None) == lib.RTN_ERR_SHAPE
    assert cabi.rtn_token_log_probs_fwd(P, 0, P, 1 << 22, 100000, F32, 3, P, P, P, P, P, P, 1 << 40, None) == lib.RTN_ERR_SHAPE  # (in pieces)
    for rows, V in ((1 << 29, 200), (1 << 27, 2000), (1 << 25, 3000)):
        assert cabi.rtn_token_log_probs_bwd(P, 0, P, P, P, P, P, P, rows, V, BF16, None) == lib.RTN_ERR_SHAPE


def test_dropout_counters_are_saved(tmp_path):
    """A training that is taken up again goes on with the masks that come next, of a model's every dropout; what was saved without them still loads."""
    m = RecurrentLanguageModel(7, 4, 2, drop_prob=0.5)
    for k, d in enumerate(m.dropouts):
        d.offset = 11 + k
    m.dropouts[2].offset = (1 << 64) - 3
    torch.save(m.state_dict(), tmp_path / "model.pt")
    state = torch.load(tmp_path / "model.pt", weights_only=True)
    other = RecurrentLanguageModel(7, 4, 2, drop_prob=0.5, seed=5)
    seeds = [d.seed for d in other.dropouts]
    other.load_state_dict(state)
    assert [d.offset for d in other.dropouts] == [11, 12, (1 << 64) - 3] and [d.seed for d in other.dropouts] == seeds
    old = {k: v for k, v in state.items() if not k.startswith("dropouts")}
    missing, unexpected = other.load_state_dict(old)
    assert not missing and not unexpected and other.dropouts[0].offset == 11
    single = Dropout(0.5)
    single.load_state_dict({})
    single.load_state_dict(Dropout(0.1).state_dict())
    assert single.offset == 0 and single.drop_prob == 0.5
    with pytest.raises(RuntimeError, match="embedding"):
        other.load_state_dict({k: v for k, v in state.items() if "embedding" not in k})


# (float64 on both sides: sums of at most a few hundred terms of about 1, each good to 2^-52)
@pytest.mark.parametrize("direction", [1, -1])
def test_recurrence_definition_against_autograd(direction):
    rng = numpy.random.default_rng(5)
    T, B, n, lens = 11, 4, 3, [11, 0, 6, 1]
    x, c0 = (torch.from_numpy(rng.normal(size=s)).requires_grad_() for s in ((T, B, 4 * n), (B, n)))
    dy, dc = rng.normal(size=(T, B, n)), rng.normal(size=(B, n))
    c, ys = c0, [None] * T
    for t in range(T) if direction > 0 else reversed(range(T)):
        z, i, f, o = x[t].chunk(4, dim=-1)
        inside = (t < torch.tensor(lens))[:, None]
        c = torch.where(inside, torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(z), c)
        ys[t] = torch.where(inside, torch.sigmoid(o) * c, 0.0)
    y = torch.stack(ys)
    want = (y, c) + torch.autograd.grad((y, c), (x, c0), (torch.from_numpy(dy), torch.from_numpy(dc)))
    a, b = x.detach().numpy(), c0.detach().numpy()
    got = ref.recurrence(a, b, lens, direction)[:2] + ref.recurrence_grad(a, dy, dc, b, lens, direction)[:2]
    for g, w in zip(got, want):
        assert numpy.abs(g - w.detach().numpy()).max() < 1e-13


def test_scores_definition_against_autograd():
    rng = numpy.random.default_rng(6)
    R, V, k = 7, 31, 5
    x = torch.from_numpy(rng.normal(size=(R, V)) * 3).requires_grad_()
    targets = torch.from_numpy(rng.integers(0, V, size=R))
    g, ge = rng.normal(size=R), rng.normal(size=R)
    log_p = torch.log_softmax(x, dim=-1)
    lp, h = log_p.gather(1, targets[:, None])[:, 0], torch.special.entr(log_p.exp()).sum(-1)
    (d,) = torch.autograd.grad((lp, h), x, (torch.from_numpy(g), torch.from_numpy(ge)))
    got = ref.scores(x.detach().numpy(), targets.numpy(), k)
    top = log_p.detach().topk(k)
    assert numpy.array_equal(got[3], top.indices.numpy())
    for a, b in ((got[0], lp), (got[1], h), (got[2], top.values), (ref.scores_grad(x.detach().numpy(), targets.numpy(), g, ge), d)):
        assert numpy.abs(a - b.detach().numpy()).max() < 1e-13


def test_closed_forms():
    """Gates that stay the same: a geometric series; logits that are all alike: log V; a mask of dropout: what is kept and its scale."""
    T, f, iz, o = 9, ref.sigmoid(0.7), ref.sigmoid(-0.4) * numpy.tanh(0.9), ref.sigmoid(0.2)
    y, c, _ = ref.recurrence(numpy.tile(numpy.array([0.9, -0.4, 0.7, 0.2]), (T, 1, 1)), [[2.0]])
    states = [f**t * 2.0 + iz * (1 - f**t) / (1 - f) for t in range(1, T + 1)]
    assert numpy.abs(y[:, 0, 0] - o * numpy.array(states)).max() < 1e-14 and abs(c[0, 0] - states[-1]) < 1e-14
    lp, h, top, ids, _ = ref.scores(numpy.full((1, 50), 3.0), [7], 2)
    assert max(abs(lp[0] + numpy.log(50)), abs(h[0] - numpy.log(50)), abs(top[0] + numpy.log(50)).max()) < 1e-14 and ids.tolist() == [[0, 1]]
    assert set(ref.keep_factors((40, 9), 0.25, 3, 4).flatten()) == {0.0, 4 / 3}
