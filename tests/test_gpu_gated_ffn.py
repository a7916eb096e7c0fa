"""gated_ffn and its gradients against 64-bit forms, with errors counted from the arithmetic (dense_util)."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from tests import dense_util as du
from tests.loss_util import assert_near
from xkernels_b200 import ops

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def no_wait_ran_out(cuda_device):
    junk = torch.full((1 << 24,), math.nan, device=cuda_device)      # what fresh tensors hold is not to be relied on
    del junk
    yield
    ops.check_status(cuda_device)


def make(M, H, I, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(1000 * seed + M + H + I)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return (n(M, H).to(dtype), (n(2 * I, H) * 1.3 / math.sqrt(H)).to(dtype), (n(H, I) / math.sqrt(I)).to(dtype), n(M, H).to(dtype))


# one row to a training batch; sizes below a tile, over a tile's edge, off every multiple; clusters that share a tile, pairs,
# several rounds of tiles
SIZES = [(1, 64, 64), (1, 7168, 2048), (3, 20000, 40), (16, 512, 136), (17, 512, 136), (2, 8, 8), (3, 65, 33), (1, 1, 1), (17, 200, 72), (64, 512, 256), (128, 1000, 136), (129, 264, 520), (200, 4096, 512),
         (257, 1024, 1416), (512, 4096, 1416), (1000, 2048, 264), (2048, 1024, 2048)]


@pytest.mark.parametrize("M,H,I", SIZES)
@pytest.mark.parametrize("dtype,limit", [(BF, None), (HF, 0.8)])
def test_forward(M, H, I, dtype, limit, cuda_device):
    x, w13, w2, _ = make(M, H, I, dtype, cuda_device)
    (want, err), (raw, eraw) = du.gated_ffn(x, w13, w2, limit)
    out, gate_up = xkb.gated_ffn(x, w13, w2, swiglu_limit=limit, save_gate_up=True)
    assert out.dtype == gate_up.dtype == dtype
    assert_near(out, want, err, "out")
    assert_near(gate_up, raw, eraw, "gate_up")
    assert torch.equal(out, xkb.gated_ffn(x, w13, w2, swiglu_limit=limit))      # the same bits again, and without gate_up


@pytest.mark.parametrize("M,H,I", SIZES)
@pytest.mark.parametrize("dtype,limit", [(BF, 0.8), (HF, None)])
def test_backward(M, H, I, dtype, limit, cuda_device):
    x, w13, w2, go = make(M, H, I, dtype, cuda_device)
    _, raw = xkb.gated_ffn(x, w13, w2, swiglu_limit=limit, save_gate_up=True)
    want = du.gated_ffn_grad(go, x, w13, w2, raw, limit)
    got = xkb.gated_ffn_backward(go, x, w13, w2, raw, swiglu_limit=limit)
    for g, (v, e), what in zip(got, want, ("x", "w13", "w2")):
        assert_near(g, v, e, "grad " + what)
    # gate and up multiplied once more: what the forward call saved, so the same bits
    again = xkb.gated_ffn_backward(go, x, w13, w2, swiglu_limit=limit)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_only_what_is_wanted(cuda_device):
    x, w13, w2, go = make(150, 256, 136, BF, cuda_device)
    _, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
    full = xkb.gated_ffn_backward(go, x, w13, w2, raw)
    for need in range(8):
        want = [bool(need >> i & 1) for i in range(3)]
        got = xkb.gated_ffn_backward(go, x, w13, w2, raw, None, *want)
        for g, f, w in zip(got, full, want):
            assert (g is None) if not w else torch.allclose(g.float(), f.float(), rtol=2.0 ** -7, atol=1e-3), need


@pytest.mark.parametrize("M", [5, 300])
def test_rows_apart_misaligned_and_turned(M, cuda_device):
    """Slices of wider tensors are read in place, tensors that no copy of the kernels can read are laid out once more."""
    H, I = 136, 72
    x, w13, w2, go = make(M, H, I, BF, cuda_device)
    want = xkb.gated_ffn(x, w13, w2), *xkb.gated_ffn_backward(go, x, w13, w2)

    def apart(t, pad):
        wide = torch.full((t.shape[0], t.shape[1] + pad), math.nan, dtype=t.dtype, device=t.device)
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    def shifted(t):
        flat = torch.full((t.numel() + 3,), math.nan, dtype=t.dtype, device=t.device)
        flat[3:] = t.reshape(-1)
        return flat[3:].view(t.shape)

    for change in (lambda t: apart(t, 8), lambda t: apart(t, 5), shifted, lambda t: t.t().contiguous().t()):
        a = [change(t) for t in (x, w13, w2, go)]
        got = xkb.gated_ffn(*a[:3]), *xkb.gated_ffn_backward(a[3], *a[:3])
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_no_rows(cuda_device):
    x, w13, w2, go = make(0, 64, 40, HF, cuda_device)
    out, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
    assert out.shape == (0, 64) and raw.shape == (0, 80)
    gx, g13, g2 = xkb.gated_ffn_backward(go, x, w13, w2, raw)
    assert gx.shape == (0, 64) and not g13.any() and not g2.any() and g13.shape == w13.shape and g2.shape == w2.shape


@pytest.mark.parametrize("M", [7, 300])
def test_nan_and_infinity_stay_in_their_rows(M, cuda_device):
    H, I = 264, 136
    x, w13, w2, go = make(M, H, I, BF, cuda_device)
    clean = xkb.gated_ffn(x, w13, w2, swiglu_limit=2.0)
    gclean = xkb.gated_ffn_backward(go, x, w13, w2, swiglu_limit=2.0)[0]
    x[3, 5], x[5, 7], go[1, 2] = math.nan, math.inf, math.nan
    out = xkb.gated_ffn(x, w13, w2, swiglu_limit=2.0)
    gx = xkb.gated_ffn_backward(go, x, w13, w2, swiglu_limit=2.0)[0]
    others = [i for i in range(M) if i not in (3, 5)]
    assert torch.equal(out[others], clean[others]) and out[3].isnan().all()
    others = [i for i in range(M) if i not in (1, 3, 5)]
    assert torch.equal(gx[others], gclean[others]) and gx[1].isnan().all() and gx[3].isnan().all()


def test_gates_far_out(cuda_device):
    """silu of large gates of both signs: neither overflows nor leaves a NaN."""
    x = torch.tensor([[80.0], [-80.0], [240.0], [-240.0], [0.0]], device=cuda_device).to(BF)
    w13, w2 = torch.ones(2, 1, device=cuda_device, dtype=BF), torch.ones(1, 1, device=cuda_device, dtype=BF)
    want = torch.nn.functional.silu(x.double()) * x.double()
    out, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
    assert_near(out, want, 2.0 ** -7 * want.abs(), "out")
    gx, _, _ = xkb.gated_ffn_backward(torch.ones_like(x), x, w13, w2, raw)
    s = torch.sigmoid(x.double())
    want = x.double() * s * (1 + x.double() * (1 - s)) + x.double() * s
    assert_near(gx, want, 2.0 ** -6 * want.abs(), "grad")


def test_limits_at_the_border(cuda_device):
    """A gate or an up exactly at the limit still has its gradient, one beyond it has none."""
    raw = torch.tensor([[2.0, 2.015625, 2.0, 2.0, -2.0, -2.015625]], device=cuda_device).to(BF)   # gates 2, 2+, 2; ups 2, -2, -2-
    x = torch.ones(1, 8, device=cuda_device, dtype=BF)
    w13, w2 = torch.ones(6, 8, device=cuda_device, dtype=BF), torch.eye(8, 3, device=cuda_device, dtype=BF)
    go = torch.ones(1, 8, device=cuda_device, dtype=BF)
    _, g13, _ = xkb.gated_ffn_backward(go, x, w13, w2, raw, swiglu_limit=2.0)
    live = (g13[:, 0] != 0).tolist()
    assert live == [True, False, True, True, True, False]


def test_two_streams_and_captured_calls(cuda_device):
    """Two calls at once share nothing; captured ones replay with new inputs, each graph with its own memory."""
    sets = [make(M, 512, 264, BF, cuda_device, seed=M) for M in (1, 64, 200, 600)]

    def step(x, w13, w2, go):
        out, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
        return out, raw, *xkb.gated_ffn_backward(go, x, w13, w2, raw, swiglu_limit=None)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        got.clear()
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(step(*s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    for _ in range(2):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    sets[2][0].neg_()
    graphs[2].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[2], step(*sets[2])))


def test_inputs_are_left_alone_and_sms_may_be_kept_free(cuda_device):
    from xkernels_b200 import _lib

    t = make(700, 1024, 520, BF, cuda_device)
    before = [a.clone() for a in t]
    want = xkb.gated_ffn(*t[:3])
    try:
        _lib.set_sm_margin(20)
        assert torch.equal(xkb.gated_ffn(*t[:3]), want)
    finally:
        _lib.set_sm_margin(0)
    assert all(torch.equal(a, b) for a, b in zip(t, before))


def test_offsets_beyond_32_bits(cuda_device):
    """2.5e9 elements of gate and up: the last rows are those of a short call with the same weights, bit for bit where the tile is
    the same and to a rounding's error where not."""
    M, H, I, tail = 1_200_000, 64, 1040, 700
    g = torch.Generator(device=cuda_device).manual_seed(9)
    x = torch.randn(M, H, generator=g, device=cuda_device, dtype=torch.float32).to(BF)
    w13, w2 = (torch.randn(2 * I, H, generator=g, device=cuda_device) / 8).to(BF), (torch.randn(H, I, generator=g, device=cuda_device) / 32).to(BF)
    out, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
    assert raw.numel() > 2 ** 31
    (want, err), (wraw, eraw) = du.gated_ffn(x[-tail:], w13, w2)
    assert_near(out[-tail:], want, err, "out")
    assert_near(raw[-tail:], wraw, eraw, "gate_up")
    go = torch.zeros_like(x)
    go[-tail:] = torch.randn(tail, H, generator=g, device=cuda_device).to(BF)        # the weights' gradients are the last rows'
    gx, g13, g2 = xkb.gated_ffn_backward(go, x, w13, w2, raw)
    del out
    (vx, ex), (v13, e13), (v2, e2) = du.gated_ffn_grad(go[-tail:], x[-tail:], w13, w2, raw[-tail:])
    assert_near(gx[-tail:], vx, ex, "grad x")
    assert_near(g13, v13, e13, "grad w13")
    assert_near(g2, v2, e2, "grad w2")
    assert not gx[:-tail].any()
