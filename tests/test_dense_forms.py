"""What the differentiable form of gated_ffn asks the operator for, without a GPU: gate and up are kept where a backward pass will
use them, and nowhere else."""

import pytest
import torch

from xkernels_b200 import autograd as xka
from xkernels_b200 import ops


@pytest.fixture
def asked(monkeypatch):
    """save_gate_up of every call."""
    seen = []

    def gated_ffn(x, w13, w2, swiglu_limit=None, save_gate_up=False):
        seen.append(save_gate_up)
        gate_up = x @ w13.t()
        gate, up = gate_up.chunk(2, dim=1)
        out = (torch.nn.functional.silu(gate) * up) @ w2.t()
        return (out, gate_up) if save_gate_up else out

    monkeypatch.setattr(ops, "gated_ffn", gated_ffn)
    return seen


def leaves(*need):
    return [torch.randn(s).requires_grad_(n) for s, n in zip(((3, 4), (10, 4), (4, 5)), need)]


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_kept_where_no_gradient_is_recorded(mode, asked):
    with mode():
        for need in ((True, True, True), (False, True, False)):
            assert not xka.gated_ffn(*leaves(*need)).requires_grad
    assert not xka.gated_ffn(*leaves(False, False, False)).requires_grad
    assert asked == [False] * 3


def test_what_is_kept_for_a_gradient(asked, monkeypatch):
    given = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)      # (asked before each backward pass; there is no GPU)
    monkeypatch.setattr(ops, "gated_ffn_backward", lambda go, x, w13, w2, gate_up, limit, *need: (
        given.append(gate_up is not None), *(torch.zeros_like(t) if n else None for t, n in zip((x, w13, w2), need)))[1:])
    for i in range(3):
        xka.gated_ffn(*leaves(*(i == j for j in range(3)))).sum().backward()
    with torch.no_grad(), torch.enable_grad():
        xka.gated_ffn(*leaves(True, True, True)).sum().backward()
    xka.gated_ffn(*leaves(True, True, True), recompute=True).sum().backward()
    assert asked == given == [True] * 4 + [False]
