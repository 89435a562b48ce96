"""
CPU-side checks of the operators of whole language models: the library loads and exports what its header declares, refusals come before
any launch, the definitions that the GPU tests compare with hold (differences, torch's autograd, closed forms).
"""

from __future__ import annotations

import ctypes
import os
import re
import subprocess

import numpy
import pytest
import torch

import _model_ref as ref
import test_generated_code as generated
from returnn_amd import build, lib, model_lib
from returnn_amd.beam_search import beam_select, reorder_states
from returnn_amd.delta_rule import DeltaRecurrence, gated_delta_rule
from returnn_amd.embedding import Embedding, embed
from returnn_amd.language_model import RecurrentLanguageModel

_root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16 = lib.DTYPE_F32, lib.DTYPE_BF16


@pytest.fixture(scope="module")
def cabi():
    if not os.path.exists(build.MODEL_LIB_PATH):
        build.build_library()
    return model_lib.load()


def test_header_symbols_are_exported(cabi):
    header = open(os.path.join(_root, "include", "rtn_model_ops.h")).read()
    declared = set(re.findall(r"^(?:int|size_t|const char\*) (rtn_[a-z0-9_]+)\(", header, re.M))
    assert declared == set(model_lib.SYMBOLS)
    for name in declared:
        assert getattr(cabi, name) is not None
    assert re.findall(r"ABI version of this header: (\d+)\.", header) == [str(model_lib.EXPECTED_ABI)]
    assert cabi.rtn_model_ops_abi_version() == model_lib.EXPECTED_ABI


def test_loader_refuses_another_abi_version(monkeypatch):
    monkeypatch.setattr(model_lib, "_lib", None)
    monkeypatch.setattr(model_lib, "EXPECTED_ABI", model_lib.EXPECTED_ABI + 1)
    with pytest.raises(lib.NativeLibraryMismatch):
        model_lib.load()


def test_the_library_is_never_built_silently(monkeypatch, tmp_path):
    monkeypatch.setattr(model_lib, "_lib", None)
    monkeypatch.setattr(build, "MODEL_LIB_PATH", str(tmp_path / "none.so"))
    with pytest.raises(lib.NativeLibraryMissing):
        model_lib.load()


def test_every_source_makes_a_build_necessary():
    for name in build.MODEL_HEADERS + [build.MODEL_SOURCE, build.MODEL_BINDING_SOURCE] + build.SEQUENCE_HEADERS:
        assert os.path.exists(os.path.join(build.CSRC_DIR, name)), name


P = 1 << 20  # an address that is never looked at: every call below is refused by the host, or has nothing to do
SHAPE, ARG, RANGE, WORKSPACE, OK = lib.RTN_ERR_SHAPE, lib.RTN_ERR_ARG, lib.RTN_ERR_RANGE, lib.RTN_ERR_WORKSPACE, lib.RTN_OK


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(T=-1), SHAPE), (dict(T=(1 << 30) + 1), SHAPE), (dict(B=-1), SHAPE), (dict(Hk=-1), SHAPE), (dict(H=-2), SHAPE), (dict(H=3), SHAPE), (dict(Hk=0), SHAPE),
        (dict(dk=0), SHAPE), (dict(dk=129), SHAPE), (dict(dv=0), SHAPE), (dict(dv=65537), SHAPE), (dict(ldq=15), SHAPE), (dict(ldk=15), SHAPE), (dict(ldv=39), SHAPE),
        (dict(dtype=2), ARG), (dict(direction=0), RANGE), (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(g=None), ARG), (dict(beta=None), ARG),
        (dict(y=None), ARG), (dict(sN=None), ARG), (dict(q=P + 1), ARG), (dict(k=P + 1), ARG), (dict(v=P + 1), ARG), (dict(y=P + 1), ARG), (dict(g=P + 2), ARG),
        (dict(beta=P + 2), ARG), (dict(s0=P + 2), ARG), (dict(sN=P + 2), ARG), (dict(lens=P + 4), ARG), (dict(saved=P + 4), ARG),
        (dict(), WORKSPACE), (dict(ws=P, bytes=16), WORKSPACE), (dict(ws=P + 4, bytes=1 << 40), ARG),
        (dict(ldq=1 << 25, ws=P, bytes=1 << 40), SHAPE), (dict(ldk=1 << 40, ws=P, bytes=1 << 40), SHAPE), (dict(ldv=1 << 25, ws=P, bytes=1 << 40), SHAPE),
        (dict(B=1 << 30, ws=P, bytes=1 << 62), SHAPE), (dict(B=1 << 30, T=3), SHAPE), (dict(B=0), OK), (dict(Hk=0, H=0), OK),
    ],
)  # fmt: skip
def test_delta_refusals(cabi, change, code):
    a = dict(q=P, ldq=0, k=P, ldk=0, v=P, ldv=0, g=P, beta=P, s0=P, lens=P, y=P, sN=P, saved=None, T=100, B=3, Hk=2, H=4, dk=8, dv=10, dtype=BF16, scale=1.0, direction=1, ws=None, bytes=0)
    a.update(change)
    assert cabi.rtn_delta_rule_fwd(*a.values(), None) == code
    assert bool(model_lib.last_error()) == (code != OK)


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(T=-1), SHAPE), (dict(H=3), SHAPE), (dict(dk=129), SHAPE), (dict(ldy=39), SHAPE), (dict(ldq=15), SHAPE), (dict(dtype=7), ARG), (dict(direction=3), RANGE),
        (dict(saved=None), ARG), (dict(dy=None), ARG), (dict(dq=None), ARG), (dict(dk_=None), ARG), (dict(dv_=None), ARG), (dict(dg=None), ARG), (dict(db=None), ARG),
        (dict(ds0=None), ARG), (dict(dy=P + 1), ARG), (dict(dq=P + 1), ARG), (dict(ds=P + 2), ARG), (dict(ds0=P + 1), ARG), (dict(), WORKSPACE),
        (dict(ws=P + 8, bytes=1 << 40), ARG), (dict(ldy=1 << 25, ws=P, bytes=1 << 40), SHAPE), (dict(B=0), OK),
    ],
)  # fmt: skip
def test_delta_gradient_refusals(cabi, change, code):
    a = dict(q=P, ldq=0, k=P, ldk=0, v=P, ldv=0, g=P, beta=P, lens=P, saved=P, dy=P, ldy=0, ds=P, dq=P, dk_=P, dv_=P, dg=P, db=P, ds0=P, T=100, B=3, Hk=2, H=4, dk=8, dv=10, dtype=BF16,
             scale=1.0, direction=1, ws=None, bytes=0)  # fmt: skip
    a.update(change)
    assert cabi.rtn_delta_rule_bwd(*a.values(), None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(), ARG), (dict(dq=P), ARG), (dict(dq=P, dk_=P + 1), ARG), (dict(dq=P, dk_=P, T=1 << 30, B=1 << 30), SHAPE), (dict(dq=P, dk_=P, Hk=(1 << 31) - 1), SHAPE),
        (dict(T=0), OK), (dict(B=0), OK), (dict(Hk=0), OK),
    ],
)  # fmt: skip
def test_delta_gradient_refusals_without_values(cabi, change, code):
    """Queries and keys without a head of values: their gradients are asked for all the same, and nothing else."""
    a = dict(q=P, ldq=0, k=P, ldk=0, v=None, ldv=0, g=None, beta=None, lens=None, saved=None, dy=None, ldy=0, ds=None, dq=None, dk_=None, dv_=None, dg=None, db=None, ds0=None, T=100, B=3, Hk=2, H=0,
             dk=8, dv=10, dtype=BF16, scale=1.0, direction=1, ws=None, bytes=0)  # fmt: skip
    a.update(change)
    assert cabi.rtn_delta_rule_bwd(*a.values(), None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(V=-1), SHAPE), (dict(V=1 << 31), SHAPE), (dict(D=-1), SHAPE), (dict(ld=4), SHAPE), (dict(dtype=9), ARG),
        (dict(tokens=None), ARG), (dict(table=None), ARG), (dict(y=None), ARG), (dict(tokens=P + 4), ARG), (dict(table=P + 1), ARG), (dict(y=P + 1), ARG),
        (dict(rows=(1 << 31) - 1, D=1 << 20), SHAPE), (dict(rows=0), OK), (dict(D=0), OK),
    ],
)  # fmt: skip
def test_embedding_refusals(cabi, change, code):
    a = dict(tokens=P, table=P, ld=0, y=P, rows=6, V=7, D=5, dtype=BF16, scale=1.0)
    a.update(change)
    assert cabi.rtn_embedding_fwd(*a.values(), None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(rows=-1), SHAPE), (dict(V=1 << 31), SHAPE), (dict(D=-1), SHAPE), (dict(ld=4), SHAPE), (dict(dtype=9), ARG), (dict(tokens=None), ARG), (dict(dy=None), ARG),
        (dict(d=None), ARG), (dict(tokens=P + 4), ARG), (dict(dy=P + 1), ARG), (dict(d=P + 1), ARG), (dict(), WORKSPACE), (dict(ws=P + 8, bytes=1 << 30), ARG),
        (dict(V=(1 << 31) - 1, D=1 << 20, ws=P, bytes=1 << 60), SHAPE), (dict(rows=(1 << 31) - 1, D=1 << 20, ws=P, bytes=1 << 60), SHAPE), (dict(V=0), OK), (dict(D=0), OK),
    ],
)  # fmt: skip
def test_embedding_gradient_refusals(cabi, change, code):
    a = dict(tokens=P, dy=P, ld=0, d=P, rows=6, V=7, D=5, dtype=BF16, scale=1.0, ws=None, bytes=0)
    a.update(change)
    assert cabi.rtn_embedding_bwd(*a.values(), None) == code


@pytest.mark.parametrize(
    "change,code",
    [
        (dict(B=-1), SHAPE), (dict(K=0), SHAPE), (dict(V=0), SHAPE), (dict(V=(1 << 26) + 1), SHAPE), (dict(K=64, V=1 << 25), SHAPE), (dict(dtype=5), ARG), (dict(beam=0), RANGE),
        (dict(beam=65), RANGE), (dict(beam=7, K=2, V=3), RANGE), (dict(end=-1), RANGE), (dict(end=20000), RANGE), (dict(ld=19999), SHAPE), (dict(scores=None), ARG),
        (dict(totals=None), ARG), (dict(out=None), ARG), (dict(sources=None), ARG), (dict(tokens=None), ARG), (dict(scores=P + 1), ARG), (dict(totals=P + 2), ARG),
        (dict(out=P + 2), ARG), (dict(sources=P + 4), ARG), (dict(tokens=P + 4), ARG), (dict(), WORKSPACE), (dict(ws=P + 8, bytes=1 << 30), ARG),
        (dict(B=1 << 30, ws=P, bytes=1 << 60), SHAPE), (dict(B=0), OK),
    ],
)  # fmt: skip
def test_beam_refusals(cabi, change, code):
    a = dict(scores=P, ld=0, totals=P, ended=P, end=3, out=P, sources=P, tokens=P, B=2, K=4, V=20000, dtype=F32, beam=5, ws=None, bytes=0)
    a.update(change)
    assert cabi.rtn_beam_select(*a.values(), None) == code


def test_reorder_refusals(cabi):
    def call(count=1, src=P, dst=P, size=8, sources=P, B=2, K=3, beam=4, lists=True):
        pointers, outs, sizes = (ctypes.c_void_p * 1)(src), (ctypes.c_void_p * 1)(dst), (ctypes.c_int64 * 1)(size)
        return cabi.rtn_reorder_rows(count, pointers if lists else None, outs, sizes, sources, B, K, beam, None)

    assert [call(count=-1), call(B=-1), call(K=-1), call(beam=-1), call(size=-1)] == [SHAPE] * 5
    assert [call(src=None), call(dst=None), call(sources=None), call(sources=P + 4), call(lists=False)] == [ARG] * 5
    assert [call(B=1 << 30, beam=1 << 10), call(size=1 << 62)] == [SHAPE] * 2
    assert [call(count=0), call(B=0), call(beam=0), call(size=0)] == [OK] * 4


def test_workspaces_of_sizes_that_are_refused_are_nothing(cabi):
    for T, B, Hk, H, dk, dv in ((-1, 2, 1, 1, 8, 8), (100, -2, 1, 1, 8, 8), (100, 2, 1, 1, 0, 8), (100, 2, 1, 1, 129, 8), (100, 2, 1, 1, 8, 0), (100, 0, 1, 1, 8, 8), (100, 2, 0, 0, 8, 8)):
        assert cabi.rtn_delta_rule_fwd_workspace_bytes(T, B, Hk, H, dk, dv, BF16, 0) == cabi.rtn_delta_rule_saved_bytes(T, B, Hk, H, dk, dv, BF16) == 0
        assert cabi.rtn_delta_rule_bwd_workspace_bytes(T, B, Hk, H, dk, dv, BF16) == 0
    assert cabi.rtn_embedding_bwd_workspace_bytes(-1, 5, 5, F32) == cabi.rtn_embedding_bwd_workspace_bytes(5, 1 << 31, 5, F32) == 0
    assert cabi.rtn_beam_select_workspace_bytes(1, 1, 0, F32, 1) == cabi.rtn_beam_select_workspace_bytes(1, 0, 5, F32, 1) == cabi.rtn_beam_select_workspace_bytes(1, 1, 100000, F32, 65) == 0


def test_cpu_tensors_and_bad_arguments_are_refused(cabi):
    q, v, g = torch.zeros((4, 2, 1, 8)), torch.zeros((4, 2, 1, 5)), torch.zeros((4, 2, 1))
    with pytest.raises(RuntimeError, match="HIP"):
        gated_delta_rule(q, q, v, g, g)
    with pytest.raises(RuntimeError, match="HIP"):
        DeltaRecurrence(5, 4)(torch.zeros((2, 3, 5)))
    with pytest.raises(RuntimeError, match="HIP"):
        embed(torch.zeros((3,), dtype=torch.int64), torch.zeros((4, 5)))
    with pytest.raises(RuntimeError, match="HIP"):
        beam_select(torch.zeros((2, 5)), torch.zeros((2,)), 2)
    with pytest.raises(RuntimeError, match="HIP"):
        reorder_states([torch.zeros((2, 5))], torch.zeros((2,), dtype=torch.int64))
    for kw in (dict(num_heads=3), dict(num_heads=0), dict(key_dim=0), dict(key_dim=129)):
        with pytest.raises(ValueError):
            DeltaRecurrence(8, 16, **kw)
    with pytest.raises(ValueError):
        DeltaRecurrence(5, 4)(torch.zeros((2, 3, 4)))
    with pytest.raises(ValueError):
        RecurrentLanguageModel(5, 4, 1, layer="other")


def test_modules():
    assert [DeltaRecurrence(4, n).num_heads for n in (64, 128, 512, 100)] == [1, 2, 8, 1]
    m = DeltaRecurrence(12, 300)
    assert (m.key_dim, m.value_dim) == (128, 300) and m.ff.shape == (2 * 128 + 300 + 2, 12)
    assert m.default_initial_state(batch_dims=(5,)).shape == (5, 1, 128, 300)
    assert (m.bias.split(m.split)[3] == -3.0).all() and m.bias.count_nonzero() == 1
    torch.manual_seed(3)
    e = Embedding(7, 5)
    torch.manual_seed(3)
    assert torch.equal(e.weight, torch.nn.Embedding(7, 5).weight)
    assert set(RecurrentLanguageModel(7, 4, 1).state_dict()) >= {"embedding.weight", "layers.0.ff", "output.weight"}


def test_no_kernel_loses_a_copy(tmp_path):
    """As for the other libraries: no value is copied between the end of a masked block and the switch back to all lanes."""
    if not os.path.exists(build.MODEL_LIB_PATH) or not os.path.exists(generated.OBJDUMP):
        pytest.skip("no library or no llvm-objdump")
    with open(build.MODEL_LIB_PATH, "rb") as f:
        objects = list(generated._code_objects(f.read()))
    assert len(objects) == 1
    path = tmp_path / "code.elf"
    path.write_bytes(objects[0])
    lines = subprocess.run([generated.OBJDUMP, "-d", str(path)], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines(keepends=True)
    assert sum("k_delta" in line for line in lines if line.endswith(">:\n")) > 0
    assert not generated.lost_copies(lines)


# ---- the definitions that the GPU tests compare with (float64 on both sides: sums of at most a few hundred terms of about 1, each good to 2^-52) ----
@pytest.mark.parametrize("direction", [1, -1])
def test_delta_definition_against_autograd(direction):
    rng = numpy.random.default_rng(5)
    T, B, Hk, H, dk, dv, lens = 9, 3, 2, 4, 5, 3, [9, 0, 4]
    shapes = ((T, B, Hk, dk), (T, B, Hk, dk), (T, B, H, dv), (T, B, H), (T, B, H), (B, H, dk, dv))
    x = [torch.from_numpy(rng.normal(size=s) * 0.5).requires_grad_() for s in shapes]
    q, k, v, g, b, s = x
    dy, ds = rng.normal(size=(T, B, H, dv)), rng.normal(size=(B, H, dk, dv))
    ys = [None] * T
    for t in range(T) if direction > 0 else reversed(range(T)):
        inside = (t < torch.tensor(lens))[:, None, None, None]
        qt, kt = (z[t].repeat_interleave(H // Hk, dim=1) for z in (q, k))
        eye = torch.eye(dk, dtype=torch.float64)
        through = torch.exp(g[t])[..., None, None] * (eye - b[t][..., None, None] * kt[..., :, None] * kt[..., None, :])
        s = torch.where(inside, through @ s + b[t][..., None, None] * kt[..., :, None] * v[t][..., None, :], s)
        ys[t] = torch.where(inside[..., 0], (qt[..., None, :] @ s)[..., 0, :] / dk**0.5, 0.0)
    y = torch.stack(ys)
    want = (y, s) + torch.autograd.grad((y, s), x, (torch.from_numpy(dy), torch.from_numpy(ds)))
    a = [z.detach().numpy() for z in x]
    got = ref.delta(*a, lens, direction)[:2] + ref.delta_grad(*a[:5], dy, ds, a[5], lens, direction)
    for i, j in zip(got, want):
        assert numpy.abs(i - j.detach().numpy()).max() < 1e-12


def test_delta_gradient_against_differences():
    rng = numpy.random.default_rng(6)
    T, B, Hk, H, dk, dv, lens = 5, 2, 1, 2, 3, 2, [5, 3]
    x = [rng.normal(size=s) * 0.5 for s in ((T, B, Hk, dk), (T, B, Hk, dk), (T, B, H, dv), (T, B, H), (T, B, H), (B, H, dk, dv))]
    dy, ds = rng.normal(size=(T, B, H, dv)), rng.normal(size=(B, H, dk, dv))
    grads = ref.delta_grad(*x[:5], dy, ds, x[5], lens)

    def value():
        y, s, _ = ref.delta(*x, lens)
        return (y * dy).sum() + (s * ds).sum()

    h = 1e-5  # (errors of h^2 and 1e-16 / h)
    for a, d in zip(x, grads):
        for at in numpy.ndindex(a.shape):
            old = a[at]
            a[at] = old + h
            up = value()
            a[at] = old - h
            down = value()
            a[at] = old
            assert abs((up - down) / (2 * h) - d[at]) < 1e-8


def test_delta_closed_forms():
    """Keys that are unit vectors: every value is stored under its own, what is written again is replaced, decay and forgetting."""
    dk, dv = 4, 3
    rng = numpy.random.default_rng(7)
    eye, v = numpy.eye(dk)[:, None, None, :], rng.normal(size=(dk, 1, 1, dv))
    one, zero = numpy.ones((dk, 1, 1)), numpy.zeros((dk, 1, 1))
    _, s, _ = ref.delta(eye, eye, v, zero, one)
    assert numpy.abs(s[0, 0] - v[:, 0, 0]).max() < 1e-15
    y, s, _ = ref.delta(eye[:1].repeat(2, 0), eye[:1].repeat(2, 0), v[:2], zero[:2], one[:2], scale=1.0)
    assert numpy.abs(s[0, 0, 0] - v[1, 0, 0]).max() < 1e-15 and numpy.abs(y[1, 0, 0] - v[1, 0, 0]).max() < 1e-15
    _, s, _ = ref.delta(eye, eye, v, numpy.full((dk, 1, 1), numpy.log(0.5)), one)
    assert numpy.abs(s[0, 0] - v[:, 0, 0] * 0.5 ** numpy.arange(dk - 1, -1, -1)[:, None]).max() < 1e-15
    _, s, _ = ref.delta(eye, eye, v, numpy.full((dk, 1, 1), -numpy.inf), one, rng.normal(size=(1, 1, dk, dv)))
    assert numpy.abs(s[0, 0, -1] - v[-1, 0, 0]).max() < 1e-15 and not s[0, 0, :-1].any()


def test_embedding_definition_against_autograd():
    rng = numpy.random.default_rng(8)
    tokens = rng.integers(0, 5, size=(6, 4))
    w = torch.from_numpy(rng.normal(size=(5, 3))).requires_grad_()
    dy = rng.normal(size=(6, 4, 3))
    y = 1.5 * torch.nn.functional.embedding(torch.from_numpy(tokens), w)
    (d,) = torch.autograd.grad(y, w, torch.from_numpy(dy))
    assert numpy.abs(ref.embed(tokens, w.detach().numpy(), 1.5) - y.detach().numpy()).max() < 1e-13
    out, most, count = ref.embed_grad(tokens, dy, 5, 1.5)
    assert numpy.abs(out - d.numpy()).max() < 1e-13 and (most >= abs(out)).all() and count.sum() == 24
    y = ref.embed([-1, 5, 2], w.detach().numpy())
    assert not y[0].any() and numpy.isnan(y[1]).all()


def test_beam_definition():
    totals, sources, tokens = ref.beam([[[1.0, 3.0, 3.0], [2.0, 0.0, 3.0]]], [[0.0, 0.0]], 4)
    assert totals.tolist() == [[3.0, 3.0, 3.0, 2.0]] and sources.tolist() == [[0, 0, 1, 1]] and tokens.tolist() == [[1, 2, 2, 0]]
    totals, sources, tokens = ref.beam([[[1.0, 3.0, 3.0], [2.0, 0.0, 3.0]]], [[-1.0, -numpy.inf]], 5, [[True, False]], 2)
    assert totals[0, 0] == -1.0 and numpy.isneginf(totals[0, 1:]).all() and sources.tolist() == [[0, 0, 0, 1, 1]] and tokens.tolist() == [[2, 0, 1, 0, 1]]
    totals, sources, tokens = ref.beam([[[1.0, numpy.nan, numpy.inf]]], [[0.5]], 3)
    assert numpy.isnan(totals[0, 0]) and totals[0, 1:].tolist() == [numpy.inf, 1.5] and tokens.tolist() == [[1, 2, 0]]
