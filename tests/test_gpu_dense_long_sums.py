"""Sums of the dense operators over very many rows, or over a very wide layer.  A tensor core cuts off at each step of 16 products: the sum
to its 24 bits and each product at the sum's last place or a little below, together less than 5 ulp (2^-23) of the sum so far.  An
accumulator takes at most 16384 products, 1024 steps, over which a sum of one sign is half its last value on average: it is off by less
than 1024 * 5 / 2 ulp.  The parts are added up with rounding, a few ulp more.  None of this grows with the number of products."""

import pytest
import torch

import xkernels_b200 as xkb
from tests.loss_util import assert_near, half_step
from xkernels_b200 import ops

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
CUT = (1024 * 5 / 2 + 64) * 2.0 ** -23


@pytest.fixture(autouse=True)
def no_wait_ran_out(cuda_device):
    yield
    ops.check_status(cuda_device)


def some(g, *shape):
    """Numbers of one sign, 0.5 .. 1.5."""
    return 0.5 + torch.rand(*shape, generator=g, device=g.device)


def by_rows(a, b):
    """a^T b in 64 bits, a piece of the rows at a time."""
    return sum(p.double().t() @ q.double() for p, q in zip(a.split(1 << 18), b.split(1 << 18)))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,H,I", [(1 << 20, 64, 64), (700_001, 72, 33), (16384 * 3 + 1, 1024, 520)])
def test_weights_of_a_block_over_many_rows(M, H, I, dtype, cuda_device):
    """gate and up, and the gradients of both, of one sign; those and silu(gate) up are rounded once (half a step)."""
    g = torch.Generator(device=cuda_device).manual_seed(M)
    gate_up, x = some(g, M, 2 * I).to(dtype), some(g, M, H).to(dtype)
    go, w2, w13 = (some(g, M, H) / 1024).to(dtype), (some(g, H, I) / H).to(dtype), torch.zeros(2 * I, H, device=cuda_device, dtype=dtype)
    got = xkb.gated_ffn_backward(go, x, w13, w2, gate_up)[1:]
    gate, up = gate_up.float().chunk(2, dim=1)
    s = torch.sigmoid(gate)
    dh = go.float() @ w2.float()
    d13 = torch.cat([dh * up * s * (1 + gate * (1 - s)), dh * gate * s], dim=1)
    w13_, w2_ = by_rows(d13, x), by_rows(go, gate * s * up)
    # the fp32 reference of an element, and the kernel's: 2^-18
    rel = half_step(dtype) + 2.0 ** -18 + CUT
    for v, t, what in ((w13_, got[0], "grad w13"), (w2_, got[1], "grad w2")):
        assert_near(t, v, v.abs() * rel, what)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_weight_of_a_head_over_many_rows(dtype, cuda_device):
    """Gradients of the logits that no label reduces: 1/V of each row's factor, which is a power of two, as are the hidden states."""
    M, H, V = 600_000, 64, 256
    x = torch.ones(M, H, device=cuda_device, dtype=dtype)
    x[:, 1::2] = 0.25
    w = torch.zeros(V, H, device=cuda_device, dtype=dtype)
    labels = torch.full((M,), V - 1, device=cuda_device)
    labels[::3] = -1
    gl = 1 + torch.rand(M, generator=torch.Generator(device=cuda_device).manual_seed(1), device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    gx, gw = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_loss=gl / 4096)
    total = (torch.where(labels >= 0, gl, 0.0).double() / 4096).sum() / V
    want = total * x[0].double().expand(V - 1, H)
    rel = half_step(dtype) + 2.0 ** -18 + CUT
    assert_near(gw[:-1], want, want * rel, "grad weight")


@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_very_wide_block(M, dtype, cuda_device):
    """Forward and the gradient of x, which are sums over the 2^18 and 2^19 columns between the products."""
    H, I = 64, 1 << 18
    g = torch.Generator(device=cuda_device).manual_seed(M)
    x, go = some(g, M, H).to(dtype), some(g, M, H).to(dtype)
    w13, w2 = (some(g, 2 * I, H) / H).to(dtype), (some(g, H, I) / H).to(dtype)
    out, gate_up = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
    gate, up = (x.double() @ w13.double().t()).chunk(2, dim=1)
    rel = half_step(dtype) + 2.0 ** -18 + CUT
    want = (gate * torch.sigmoid(gate) * up) @ w2.double().t()
    assert_near(out, want, want * rel, "out")
    all_of_them = xkb.gated_ffn_backward(go, x, w13, w2, gate_up)
    alone = xkb.gated_ffn_backward(go, x, w13, w2, gate_up, need_grad_w13=False, need_grad_w2=False)
    gate, up = gate_up.double().chunk(2, dim=1)
    s = torch.sigmoid(gate)
    dh = go.double() @ w2.double()
    want = torch.cat([dh * up * s * (1 + gate * (1 - s)), dh * gate * s], dim=1) @ w13.double()
    assert_near(all_of_them[0], want, want * rel, "grad x")
    assert_near(alone[0], want, want * rel, "grad x alone")


def test_hidden_states_over_a_large_vocabulary(cuda_device):
    """grad_hidden is a sum over the vocabulary: equal probabilities, a power of two and exact in fp16, and weights of one sign."""
    M, H, V = 260, 4096, 1 << 18
    g = torch.Generator(device=cuda_device).manual_seed(2)
    w = torch.empty(V, H, dtype=HF, device=cuda_device)
    for part in w.split(1 << 14):
        part.copy_(some(g, *part.shape))
    x, labels = torch.zeros(M, H, device=cuda_device, dtype=HF), torch.zeros(M, dtype=torch.int64, device=cuda_device)
    r = xkb.linear_cross_entropy(x, w, labels)
    gx, _ = xkb.linear_cross_entropy_backward(x, w, labels, r.stats, grad_lse=torch.full((M,), 64.0, device=cuda_device))
    want = (64 / V * w.sum(dim=0, dtype=torch.float64)).expand(M, H)
    assert_near(gx, want, want * (2.0 ** -18 + CUT), "grad hidden")
