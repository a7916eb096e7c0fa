"""Gradients of up to 16 rows, whose operands between the products have two terms of their type: what is left is the products' fp32 and the
result's own rounding, and second terms add to the right rows."""

import pytest
import torch

import xkernels_b200 as xkb
from tests import dense_util as du
from tests.loss_util import assert_near, half_step
from tests.test_gpu_gated_ffn import BF, HF, no_wait_ran_out  # noqa: F401
from tests.test_gpu_gated_ffn import make as make_block
from tests.test_gpu_linear_cross_entropy import make as make_head

pytestmark = pytest.mark.gpu

ROWS = [1, 2, 3, 7, 8, 9, 15, 16]


def twice(x, err, dtype):
    """How far x, known to err, is off in two terms of dtype: half a step of the first one's half step (fp16: of the smallest number's, 2^-25)."""
    return err + half_step(dtype) ** 2 * 1.01 * (x.abs() + err) + (2.0 ** -25 if dtype == HF else 2.0 ** -126)


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("H,I", [(1552, 392), (264, 1001), (65, 33), (4096, 1416)])
@pytest.mark.parametrize("dtype,limit", [(BF, None), (HF, 0.8)])
def test_block(M, H, I, dtype, limit, cuda_device):
    x, w13, w2, go = make_block(M, H, I, dtype, cuda_device)
    _, raw = xkb.gated_ffn(x, w13, w2, swiglu_limit=limit, save_gate_up=True)
    got = xkb.gated_ffn_backward(go, x, w13, w2, raw, swiglu_limit=limit)
    again = xkb.gated_ffn_backward(go, x, w13, w2, swiglu_limit=limit)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    X, W13, W2, GO, RAW = (t.double() for t in (x, w13, w2, go, raw))
    gate, up = du.clamped(RAW, limit)
    open_gate, open_up = (RAW[:, :I] <= limit, RAW[:, I:].abs() <= limit) if limit else (1.0, 1.0)
    s = torch.sigmoid(gate)
    dh, edh = du.product(GO, torch.zeros_like(GO), W2.t())
    a, b, h = up * s * (1 + gate * (1 - s)) * open_gate, gate * s * open_up, gate * s * up
    ea, eb = 2.0 ** -19 * up.abs() * s * (1 + gate.abs()), 2.0 ** -20 * (gate * s).abs()
    d13 = torch.cat([dh * a, dh * b], dim=1)
    e13 = torch.cat([edh * (a.abs() + ea) + dh.abs() * ea, edh * (b.abs() + eb) + dh.abs() * eb], dim=1)
    e13, eh = twice(d13, e13, dtype), twice(h, 2.0 ** -20 * h.abs(), dtype)
    g2, e2 = du.product(h.t().contiguous(), eh.t().contiguous(), GO.t())
    want = (du.product(d13, e13, W13.t()), du.product(d13.t().contiguous(), e13.t().contiguous(), X.t()), (g2.t(), e2.t()))
    for t, (v, e), what in zip(got, want, ("x", "w13", "w2")):
        assert_near(t, v, e, "grad " + what)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        alone = xkb.gated_ffn_backward(go, x, w13, w2, raw, limit, *need)
        for t, (v, e), n in zip(alone, want, need):
            assert (t is not None) == n
            if n:
                assert_near(t, v, e, "alone")


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("H,V", [(136, 25212), (376, 1077), (65, 2), (2056, 3201), (4096, 70001)])
@pytest.mark.parametrize("dtype,padding", [(BF, 0.0), (HF, 0.4)])
def test_head(M, H, V, dtype, padding, cuda_device):
    x, w, labels = make_head(M, H, V, dtype, cuda_device, padding)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    gl, gs = torch.randn(M, generator=g, device=cuda_device), 0.1 * torch.randn(M, generator=g, device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    got = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl, grad_lse=gs)
    scale = du.scale_of(dtype, labels, gl, gs)
    on = labels >= 0
    X, W = torch.where(on[:, None], x, torch.zeros_like(x)).double(), w.double()
    z, ez = du.product(X, torch.zeros_like(X), W)
    e = z - r.stats[:, :1].double() - r.stats[:, 1:].double()
    own = torch.zeros_like(z).scatter_(1, labels.long().clamp(min=0)[:, None], gl.double()[:, None])
    p = e.exp() * (gl.double() + gs.double())[:, None]
    d = torch.where(on[:, None], p - own, 0.0)
    ed = p.abs() * (ez + 2.0 ** -20 + du.U23 * (z.abs() + e.abs())) + 2.0 ** -22 * (p.abs() + own.abs())
    ed = torch.where(on[:, None], twice(d * scale, ed * scale, dtype) / scale, 0.0)
    want = du.product(d, ed, W.t()), du.product(d.t().contiguous(), ed.t().contiguous(), X.t())
    for t, (v, e), what in zip(got, want, ("hidden", "weight")):
        assert_near(t, v, e, "grad " + what)
    for need in ((True, False), (False, True)):
        alone = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, gl, gs, *need)
        for t, (v, e), n in zip(alone, want, need):
            assert (t is not None) == n
            if n:
                assert_near(t, v, e, "alone")
    assert not got[0][~on].any()
