"""linear_cross_entropy and its gradients against 64-bit forms, with errors counted from the arithmetic (dense_util)."""

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


def make(M, H, V, dtype, dev, padding=0.0, seed=0):
    g = torch.Generator(device=dev).manual_seed(1000 * seed + M + H + V)
    w = (torch.randn(V, H, generator=g, device=dev) * 1.5 / math.sqrt(H)).to(dtype)
    labels = torch.randint(0, V, (M,), generator=g, device=dev)
    x = torch.randn(M, H, generator=g, device=dev) + 3 * torch.rand(M, 1, generator=g, device=dev) * w[labels].float()
    labels[torch.rand(M, generator=g, device=dev) < padding] = -100
    return x.to(dtype), w, labels


def stats_near(r, x, w, labels):
    loss, lse, m, l, err = du.cross_entropy(x, w, labels)
    for got, want, what in ((r.loss, loss, "loss"), (r.lse, lse, "lse"), (r.stats[:, 0], m, "m"), (r.stats[:, 1], l, "l")):
        assert_near(got, want, err, what)


SIZES = [(1, 64, 1000), (1, 4096, 5003), (2, 8, 1), (3, 65, 2), (1, 1, 7), (5, 72, 129), (64, 512, 5001), (77, 2056, 3201), (128, 136, 255), (129, 264, 640),
         (300, 1000, 5003), (520, 2048, 3000), (1100, 640, 32001)]


@pytest.mark.parametrize("M,H,V", SIZES)
@pytest.mark.parametrize("dtype,padding", [(BF, 0.0), (HF, 0.4)])
def test_forward(M, H, V, dtype, padding, cuda_device):
    x, w, labels = make(M, H, V, dtype, cuda_device, padding)
    r = xkb.linear_cross_entropy(x, w, labels)
    stats_near(r, x, w, labels)
    again = xkb.linear_cross_entropy(x, w, labels.to(torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(r, again))       # the same bits, from 32-bit labels too


@pytest.mark.parametrize("M,H,V", SIZES)
@pytest.mark.parametrize("dtype,padding", [(BF, 0.4), (HF, 0.0)])
def test_backward(M, H, V, dtype, padding, cuda_device):
    x, w, labels = make(M, H, V, dtype, cuda_device, padding)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    gl, gs = torch.randn(M, generator=g, device=cuda_device), 0.1 * torch.randn(M, generator=g, device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    for a, b in ((gl, None), (gl, gs), (None, gs)):
        want = du.cross_entropy_grad(x, w, labels, r.stats, a, b, du.scale_of(dtype, labels, a, b))
        got = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=a, grad_lse=b)
        for t, (v, e), what in zip(got, want, ("hidden", "weight")):
            assert_near(t, v, e, "grad " + what)
    again = xkb.linear_cross_entropy_backward(x, w, labels.to(torch.int32), r.stats, grad_lse=gs)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("M,H,V", [(2048, 64, 70001), (300, 128, 70001)])
def test_pieces_of_the_vocabulary_and_parts_of_it(M, H, V, cuda_device):
    """More of the logits' gradient than is held at a time; a hidden state's gradient added up in parts."""
    x, w, labels = make(M, H, V, BF, cuda_device, 0.2)
    gl = torch.rand(M, device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    want = du.cross_entropy_grad(x, w, labels, r.stats, gl, None)
    got = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl)
    for t, (v, e), what in zip(got, want, ("hidden", "weight")):
        assert_near(t, v, e, "grad " + what)
    only_x = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl, need_grad_weight=False)
    only_w = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl, need_grad_hidden=False)
    assert only_x[1] is None and only_w[0] is None
    assert_near(only_x[0], *want[0], "grad hidden alone")
    assert_near(only_w[1], *want[1], "grad weight alone")


@pytest.mark.parametrize("M", [6, 400])
def test_padding_rows_are_not_read(M, cuda_device):
    H, V = 264, 1003
    x, w, labels = make(M, H, V, BF, cuda_device, 0.5)
    labels[:2] = torch.tensor([-1, 5], device=cuda_device)
    off = labels < 0
    gl = torch.rand(M, device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    want = *r, *xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl, grad_lse=gl)
    x2, gl2, st2 = x.clone(), gl.clone(), r.stats.clone()
    x2[off] = math.nan
    gl2[off] = math.inf
    st2[off] = math.nan
    got = *xkb.linear_cross_entropy(x2, w, labels), *xkb.linear_cross_entropy_backward(x2, w, labels, st2, grad_loss=gl2, grad_lse=gl2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not r.loss[off].any() and not r.lse[off].any() and not r.stats[off].any() and not want[3][off].any()


@pytest.mark.parametrize("M", [4, 300])
def test_no_label_at_all_and_no_rows(M, cuda_device):
    x, w, _ = make(M, 72, 333, HF, cuda_device)
    labels = torch.full((M,), -1, device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    assert not r.loss.any() and not r.lse.any() and not r.stats.any()
    gx, gw = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=torch.ones(M, device=cuda_device))
    assert not gx.any() and not gw.any() and gx.shape == x.shape and gw.shape == w.shape
    r = xkb.linear_cross_entropy(x[:0], w, labels[:0])
    assert r.loss.shape == (0,) and r.stats.shape == (0, 2)
    gx, gw = xkb.linear_cross_entropy_backward(x[:0], w, labels[:0], r.stats, grad_loss=r.loss)
    assert gx.shape == (0, 72) and not gw.any()


@pytest.mark.parametrize("M", [6, 300])
def test_labels_outside_nan_and_infinity(M, cuda_device):
    H, V = 136, 500
    x, w, labels = make(M, H, V, BF, cuda_device)
    clean = xkb.linear_cross_entropy(x, w, labels)
    labels[1], labels[2] = V, 2 ** 40
    x[3, 0], x[4, 1] = math.nan, math.inf
    r = xkb.linear_cross_entropy(x, w, labels)
    rest = [i for i in range(M) if i not in (1, 2, 3, 4)]
    assert torch.equal(r.loss[rest], clean.loss[rest]) and r.loss[1:5].isnan().all() and r.lse[3:5].isnan().all()
    assert torch.equal(r.lse[1:3], clean.lse[1:3])           # the label has no part in it
    gl = torch.ones(M, device=cuda_device)
    gx, _ = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl, need_grad_weight=False)
    assert gx[1:5].isnan().all() and gx[rest].isfinite().all()


def test_logits_far_apart(cuda_device):
    """One logit far above the rest, all equal, and very negative ones: sums hold, probabilities of 0 stay 0."""
    V = 1000
    w = torch.zeros(V, 8, device=cuda_device, dtype=BF)
    w[7, 0], w[:, 1], w[11, 2] = 1, -1, 1
    x = torch.zeros(4, 8, device=cuda_device, dtype=BF)
    x[0, 0], x[1, 1], x[2, 2], x[3, 0] = 30000.0, 30000.0, -30000.0, 10.0
    labels = torch.tensor([7, 3, 11, 8], device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    far = float(x[0, 0])      # 30000 has more bits than bf16: 234.375 * 128 is held as 234 * 128
    assert far == 29952.0
    want = [0.0, math.log(V), far + math.log(V - 1), math.log(math.exp(10.0) + V - 1)]
    assert torch.allclose(r.loss.double().cpu(), torch.tensor(want, dtype=torch.float64), rtol=1e-6, atol=1e-6)
    gx, gw = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=torch.ones(4, device=cuda_device))
    assert gx.isfinite().all() and gw.isfinite().all() and not gx[0].any()


def test_small_probabilities_in_fp16(cuda_device):
    """Gradients of a mean loss over a large vocabulary lie below fp16's smallest step; d is scaled before it is rounded."""
    M, H, V = 40, 64, 60000
    x, w, labels = make(M, H, V, HF, cuda_device)
    for size in (1.0, 1e-3, 300.0):
        gl = torch.full((M,), size, device=cuda_device)
        r = xkb.linear_cross_entropy(x, w, labels)
        (vx, ex), (vw, ew) = du.cross_entropy_grad(x, w, labels, r.stats, gl, None, du.scale_of(HF, labels, gl, None))
        gx, gw = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl)
        assert_near(gx, vx, ex, "grad hidden")
        assert_near(gw, vw, ew, "grad weight")


@pytest.mark.parametrize("M", [5, 300])
def test_rows_apart_misaligned_and_broadcast(M, cuda_device):
    H, V = 136, 777
    x, w, labels = make(M, H, V, BF, cuda_device, 0.2)
    gl = torch.rand(M, device=cuda_device)

    def step(x, w, labels, gl):
        r = xkb.linear_cross_entropy(x, w, labels)
        return *r, *xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl)

    want = step(x, w, labels, gl)

    def apart(t, pad):
        wide = torch.full((t.shape[0], t.shape[1] + pad), math.nan, dtype=t.dtype, device=t.device)
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    def shifted(t):
        flat = torch.full((t.numel() + 3,), math.nan, dtype=t.dtype, device=t.device)
        flat[3:] = t.reshape(-1)
        return flat[3:].view(t.shape)

    for change in (lambda t: apart(t, 8), lambda t: apart(t, 3), shifted, lambda t: t.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(step(change(x), change(w), labels, gl), want))
    every = torch.stack([labels, labels], dim=1)[:, 0]
    assert all(torch.equal(a, b) for a, b in zip(step(x, w, every, gl), want))
    one = torch.ones((), device=cuda_device).expand(M)           # what a sum's gradient is
    assert all(torch.equal(a, b) for a, b in zip(step(x, w, labels, one), step(x, w, labels, one.contiguous())))
    row = x[:1].expand(M, H)                                     # rows that are one and the same
    assert all(torch.equal(a, b) for a, b in zip(step(row, w, labels, gl), step(row.contiguous(), w, labels, gl)))


def test_it_is_the_loss_of_the_logits(cuda_device):
    """Beside token_logprobs of the logits, which a product in fp32 made."""
    x, w, labels = make(90, 256, 2000, BF, cuda_device, 0.3)
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        z = x.float() @ w.float().t()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    a, b = xkb.linear_cross_entropy(x, w, labels), xkb.token_logprobs(z, labels)
    err = du.cross_entropy(x, w, labels)[-1].float()
    assert bool(((a.loss + b.logprobs).abs() <= 4 * err + 1e-6).all())


def test_two_streams_and_captured_calls(cuda_device):
    sets = [(*make(M, 256, V, BF, cuda_device, 0.25, seed=V), torch.rand(M, device=cuda_device)) for M, V in ((1, 3000), (70, 1000), (500, 5000))]

    def step(x, w, labels, gl):
        r = xkb.linear_cross_entropy(x, w, labels)
        return *r, *xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
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
    sets[2][2][:] = torch.where(sets[2][2] < 0, 3, -1)           # other rows are padding now
    graphs[2].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[2], step(*sets[2])))


def test_many_rows(cuda_device):
    """Far more rows than blocks, most of them padding, and a piece of the least width."""
    M, H, V = 700_001, 64, 700
    g = torch.Generator(device=cuda_device).manual_seed(4)
    x = torch.randn(M, H, generator=g, device=cuda_device).to(BF)
    w = (torch.randn(V, H, generator=g, device=cuda_device) / 6).to(BF)
    labels = torch.randint(0, V, (M,), generator=g, device=cuda_device)
    labels[torch.rand(M, generator=g, device=cuda_device) < 0.99] = -1
    on = labels >= 0
    r = xkb.linear_cross_entropy(x, w, labels)
    few = xkb.LinearCrossEntropy(*(t[on] for t in r))
    stats_near(few, x[on], w, labels[on])
    assert not r.loss[~on].any() and not r.stats[~on].any()
    gl = torch.rand(M, generator=g, device=cuda_device)
    gx, gw = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl)
    (vx, ex), (vw, ew) = du.cross_entropy_grad(x[on], w, labels[on], few.stats, gl[on], None)
    assert_near(gx[on], vx, ex, "grad hidden")
    assert_near(gw, vw, ew, "grad weight")
    assert not gx[~on].any()
