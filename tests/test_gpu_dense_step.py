"""The dense operators with the routed ones, as a training step and a decode loop use them: a layer of routed and shared experts, a
head, the losses, backward; a captured step; leaves that need no gradient."""

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import autograd as xka
from xkernels_b200 import synth

pytestmark = pytest.mark.gpu


def model(dev, dtype, M=96, D=64, I=72, E=8, k=2, V=500):
    g = torch.Generator(device=dev).manual_seed(21)
    n = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=torch.float64) / s[-1] ** 0.5  # noqa: E731
    p = {"gate": n(E, D), "experts": n(E, D, D), "w13": 1.5 * n(2 * I, D), "w2": n(D, I), "head": 3 * n(V, D)}
    x = 6 * n(M, D)
    labels = torch.randint(0, V, (M,), generator=g, device=dev)
    mask = torch.rand(M, generator=g, device=dev) < 0.7
    return {a: b.to(dtype) for a, b in p.items()}, x.to(dtype), torch.where(mask, labels, -1), mask, k


def step(p, x, labels, mask, k, own, recompute=False):
    """cross entropy with a penalty on the log-sum-exp, and a balance loss, of a layer with routed experts and a shared one"""
    logits = x.float() @ p["gate"].float().t() if own else x @ p["gate"].t()
    if own:
        w, at = xka.topk_softmax(logits, k)
    else:
        prob = torch.softmax(logits, dim=1)
        at = torch.sort(prob, dim=1, descending=True, stable=True).indices[:, :k]
        w = prob.gather(1, at)
        w = w / w.sum(dim=1, keepdim=True)
    y = torch.tanh(torch.einsum("md,mkfd->mkf", x, p["experts"][at.long()]))
    if own:
        h = x + xka.moe_sum_reduce(y.contiguous(), w) + xka.gated_ffn(x, p["w13"], p["w2"], 4.0, recompute)
        r = xka.linear_cross_entropy(h, p["head"], labels)
        bal = xka.moe_balance_loss(logits, at, mask).loss
        loss, lse = r.loss, r.lse
    else:
        gate, up = (x @ p["w13"].t()).chunk(2, dim=1)
        act = torch.nn.functional.silu(gate.clamp(max=4.0)) * up.clamp(-4.0, 4.0)
        h = x + (w[:, :, None] * y).sum(dim=1) + act @ p["w2"].t()
        z = h @ p["head"].t()
        lse = torch.where(mask, torch.logsumexp(z, dim=1), 0.0)
        loss = torch.where(mask, lse - z.gather(1, labels.clamp(min=0)[:, None])[:, 0], 0.0)
        E = logits.shape[1]
        f = torch.bincount(at[mask].reshape(-1), minlength=E).to(x.dtype) / (k * mask.sum())
        bal = E * (f * torch.softmax(logits, dim=1)[mask].mean(dim=0)).sum()
    n = mask.sum()
    return loss.sum() / n + 1e-3 * (lse ** 2).sum() / n + 0.01 * bal


@pytest.mark.parametrize("recompute", [False, True])
def test_a_training_step_against_64_bits(recompute, cuda_device):
    """Gradients of every weight against torch's in 64 bits of the same bf16 weights.  A value passes at most eight roundings to bf16
    (x, y, h, act, d and their gradients), 2^-9 each in the norm where they do not line up: 2^-5 of a gradient's norm is far above their
    sum.  (The 64-bit form takes the same experts: logits of the gate are fp32 products of bf16 numbers.)"""
    p, x, labels, mask, k = model(cuda_device, torch.bfloat16)
    got = {n: t.clone().requires_grad_() for n, t in p.items()}
    want = {n: t.double().requires_grad_() for n, t in p.items()}
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        a, b = step(got, x, labels, mask, k, True, recompute), step(want, x.double(), labels, mask, k, False)
        a.backward()
        b.backward()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    assert abs(float(a.detach()) - float(b.detach())) <= 2.0 ** -6 * abs(float(b.detach()))
    for n in p:
        g, w = got[n].grad.double(), want[n].grad
        assert float((g - w).norm()) <= 2.0 ** -5 * float(w.norm()), n


def test_leaves_that_need_no_gradient(cuda_device):
    p, x, labels, _, _ = model(cuda_device, torch.bfloat16)
    for need in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, p["w13"], p["w2"]))]
        out = xka.gated_ffn(*leaves)
        out.float().sum().backward()
        assert [t.grad is not None for t in leaves] == [bool(need >> i & 1) for i in range(3)]
    for need in range(1, 4):
        leaves = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, p["head"]))]
        r = xka.linear_cross_entropy(*leaves, labels)
        assert not r.stats.requires_grad
        (r.loss.mean() if need != 2 else r.lse.sum()).backward()
        assert [t.grad is not None for t in leaves] == [bool(need >> i & 1) for i in range(2)]
    assert not xka.gated_ffn(x, p["w13"], p["w2"]).requires_grad
    with torch.no_grad():
        assert not xka.linear_cross_entropy(x.clone().requires_grad_(), p["head"], labels).loss.requires_grad


def test_the_differentiable_forms_refuse_capture(cuda_device, monkeypatch):
    p, x, labels, _, _ = model(cuda_device, torch.bfloat16)
    leaf = x.clone().requires_grad_()
    outs = [xka.gated_ffn(leaf, p["w13"], p["w2"]), xka.linear_cross_entropy(leaf, p["head"], labels).loss]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        xka.gated_ffn(x, p["w13"], p["w2"])            # nothing is recorded for a gradient
        for call in (lambda: xka.gated_ffn(leaf, p["w13"], p["w2"]), lambda: xka.linear_cross_entropy(leaf, p["head"], labels)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    # (the answer of a capturing stream is put in its place: a captured backward pass is not started)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for out in outs:
        with pytest.raises(RuntimeError, match="captured"):
            out.float().sum().backward()


def test_a_decode_layer_in_a_graph(cuda_device):
    """A decode step of routed INT4 experts beside the shared one, captured and replayed with new tokens."""
    c = {a: (t.to(cuda_device) if isinstance(t, torch.Tensor) else t)
         for a, t in synth.make_int4(synth.Int4Config("dense_step", M=16, K=512, N=512, E=8, top_k=2), seed=5).items()}
    g = torch.Generator(device=cuda_device).manual_seed(6)
    w13, w2 = (torch.randn(s, generator=g, device=cuda_device).to(torch.bfloat16) / 20 for s in ((528, 512), (512, 264)))
    head = torch.randn(1000, 512, generator=g, device=cuda_device).to(torch.bfloat16) / 20
    x, labels = c["A"].clone(), torch.arange(16, device=cuda_device)

    def layer():
        h = xkb.fused_moe_int4_w4a16(x, c["packed"], c["scale"], c["topk_ids"], c["topk_w"]) + xkb.gated_ffn(x, w13, w2)
        return h, xkb.linear_cross_entropy(h, head, labels).loss

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for _ in range(2):
        x.copy_(torch.randn(16, 512, generator=g, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, layer()))
