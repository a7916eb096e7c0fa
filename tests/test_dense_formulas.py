"""The 64-bit gradients that the dense kernels are compared with, against torch's and against differences (no GPU needed)."""

import pytest
import torch

from tests import dense_util


def directional(f, inputs, grads, eps=1e-5):
    """The derivative along a random direction, by differences and by the gradients."""
    g = torch.Generator().manual_seed(3)
    dirs = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in inputs]
    up, down = f(*(t + eps * d for t, d in zip(inputs, dirs))), f(*(t - eps * d for t, d in zip(inputs, dirs)))
    return float((up - down) / (2 * eps)), float(sum((a * d).sum() for a, d in zip(grads, dirs)))


@pytest.mark.parametrize("limit", [None, 0.7])
def test_gated_ffn(limit):
    g = torch.Generator().manual_seed(1)
    x, w13, w2, go = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 6), (14, 6), (6, 7), (5, 6)))

    def f(x, w13, w2):
        gate, up = dense_util.clamped(x @ w13.t(), limit)
        return ((torch.nn.functional.silu(gate) * up) @ w2.t() * go).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    f(*leaves).backward()
    got = [v for v, _ in dense_util.gated_ffn_grad(go, x, w13, w2, x @ w13.t(), limit)]
    for a, b in zip(got, leaves):
        assert torch.allclose(a, b.grad, rtol=1e-12, atol=1e-12)
    if limit is None:      # (with one, a difference may step over a corner)
        by_difference, by_gradient = directional(f, [x, w13, w2], got)
        assert abs(by_difference - by_gradient) <= 1e-6 * max(1.0, abs(by_gradient))


def test_cross_entropy():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(6, 5, generator=g, dtype=torch.float64), torch.randn(9, 5, generator=g, dtype=torch.float64)
    labels = torch.tensor([0, 8, -1, 3, 3, -7])
    a, b = torch.randn(6, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    on = labels >= 0

    def f(x, w):
        z = x @ w.t()
        lse = torch.logsumexp(z, dim=1)
        return torch.where(on, a * (lse - z.gather(1, labels.clamp(min=0)[:, None])[:, 0]) + b * lse, 0.0).sum()

    loss, lse, m, l, _ = dense_util.cross_entropy(x, w, labels)
    z = x @ w.t()
    assert torch.allclose(loss[on], torch.nn.functional.cross_entropy(z[on], labels[on], reduction="none"))
    assert torch.allclose(lse[on], torch.logsumexp(z[on], dim=1)) and torch.allclose(m + l, lse) and not loss[~on].any()
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    f(*leaves).backward()
    (gx, _), (gw, _) = dense_util.cross_entropy_grad(x, w, labels, torch.stack([m, l], dim=1), a, b)
    assert torch.allclose(gx, leaves[0].grad) and torch.allclose(gw, leaves[1].grad)
    by_difference, by_gradient = directional(f, [x, w], [gx, gw])
    assert abs(by_difference - by_gradient) <= 1e-6 * max(1.0, abs(by_gradient))
