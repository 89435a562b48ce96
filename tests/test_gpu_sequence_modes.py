"""The sequence operators in torch's modes that are not plain calls: forward derivatives, autocast regions, recomputed segments, recorded steps."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from _gpu_util import announce
from returnn_amd.dropout import dropout
from returnn_amd.recurrence import gated_recurrence
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
