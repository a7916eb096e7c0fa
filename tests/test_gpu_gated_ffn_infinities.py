"""Infinities and NaN in operands of the gated block that go into products of two terms (up to 16 rows), beside calls of more rows, which have
one: an infinite sum stays infinite, with its sign, and what such an element does not reach stays finite."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from tests.test_gpu_gated_ffn import BF, HF, no_wait_ran_out  # noqa: F401

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def some(g, *shape):
    """Numbers of one sign, 0.5 .. 1.5."""
    return 0.5 + torch.rand(*shape, generator=g, device=g.device)


def check(got, at, value, what):
    """got is `value` (an infinity or NaN) in the places `at` and finite elsewhere."""
    assert torch.equal(torch.isfinite(got), ~at.expand_as(got)), what
    if value == value:
        assert (got[at.expand_as(got)] == value).all(), what
    else:
        assert got[at.expand_as(got)].isnan().all(), what


@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 40])
@pytest.mark.parametrize("H,I", [(520, 264), (65, 33), (7168, 2048)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_gradient_of_the_output(M, H, I, dtype, value, cuda_device):
    """gate, up, weights and x of one sign: dh is `value` in row r alone, and so are both gradients there."""
    g = torch.Generator(device=cuda_device).manual_seed(M)
    x, gate_up, go = some(g, M, H).to(dtype), some(g, M, 2 * I).to(dtype), some(g, M, H).to(dtype)
    w13, w2 = (some(g, 2 * I, H) / H).to(dtype), (some(g, H, I) / H).to(dtype)
    r, h = M // 2, H // 3
    go[r, h] = value
    for saved in (gate_up, None):
        gx, g13, g2 = xkb.gated_ffn_backward(go, x, w13, w2, saved)
        rows, cols = torch.arange(M, device=cuda_device) == r, torch.arange(H, device=cuda_device) == h
        check(gx, rows[:, None], value, "grad x")
        check(g13, torch.ones(1, 1, dtype=torch.bool, device=cuda_device), value, "grad w13")
        check(g2, cols[:, None], value, "grad w2")


@pytest.mark.parametrize("M", [1, 5, 16, 17])
@pytest.mark.parametrize("H,I", [(520, 264), (65, 33), (7168, 2048)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_a_weight(M, H, I, dtype, value, cuda_device):
    """A weight of the second product, in the result; one of the first, in the gradient of x (with gate and up given)."""
    g = torch.Generator(device=cuda_device).manual_seed(M)
    x, gate_up, go = some(g, M, H).to(dtype), some(g, M, 2 * I).to(dtype), some(g, M, H).to(dtype)
    w13, w2 = (some(g, 2 * I, H) / H).to(dtype), (some(g, H, I) / H).to(dtype)
    h, i = H // 3, I // 2
    cols = torch.arange(H, device=cuda_device) == h
    bad = w2.clone()
    bad[h, i] = value
    check(xkb.gated_ffn(x, w13, bad), cols, value, "out")
    for row in (i, I + i):
        bad = w13.clone()
        bad[row, h] = value
        for others in (True, False):
            gx = xkb.gated_ffn_backward(go, x, bad, w2, gate_up, need_grad_w13=others, need_grad_w2=others)[0]
            check(gx, cols, value, "grad x")


@pytest.mark.parametrize("M", [1, 5, 16, 17])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_a_row(M, dtype, value, cuda_device):
    """An element of x, with gate and up given: it is in the gradient of the first weights alone."""
    g = torch.Generator(device=cuda_device).manual_seed(M)
    H, I = 520, 264
    x, gate_up, go = some(g, M, H).to(dtype), some(g, M, 2 * I).to(dtype), some(g, M, H).to(dtype)
    w13, w2 = (some(g, 2 * I, H) / H).to(dtype), (some(g, H, I) / H).to(dtype)
    h = H // 3
    x[M - 1, h] = value
    gx, g13, g2 = xkb.gated_ffn_backward(go, x, w13, w2, gate_up)
    check(g13, torch.arange(H, device=cuda_device) == h, value, "grad w13")
    assert torch.isfinite(gx).all() and torch.isfinite(g2).all()
