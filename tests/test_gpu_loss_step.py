"""The operators together, as a training step and a serving loop use them: a routed layer with a head, its two losses, backward;
captured steps; other streams; calls in turn that share nothing."""

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import autograd as xka

pytestmark = pytest.mark.gpu


def model(dev, dtype=torch.float32, M=48, D=32, E=12, k=3, V=300):
    g = torch.Generator(device=dev).manual_seed(11)
    n = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=torch.float64) / s[-1] ** 0.5  # noqa: E731
    p = {"gate": n(E, D), "experts": n(E, D, D), "head": n(V, D) * 4}
    x = n(M, D) * 6
    mask = torch.rand(M, generator=g, device=dev) < 0.8
    ids = torch.randint(0, V, (M,), generator=g, device=dev)
    return {a: b.to(dtype) for a, b in p.items()}, x.to(dtype), torch.where(mask, ids, -1), mask, k


def step(p, x, ids, mask, k, own):
    """loss of a routed layer with a residual and a head: -logprob + 0.01 * balance - 0.02 * entropy - 0.1 * top alternatives"""
    logits = x @ p["gate"].t()
    if own:
        w, at = xka.topk_softmax(logits, k)
    else:
        prob = torch.softmax(logits, dim=1)
        at = torch.sort(prob, dim=1, descending=True, stable=True).indices[:, :k]
        w = prob.gather(1, at)
        w = w / w.sum(dim=1, keepdim=True)
    y = torch.tanh(torch.einsum("md,mkfd->mkf", x, p["experts"][at.long()]))
    h = x + (xka.moe_sum_reduce(y.contiguous(), w, 1.5) if own else 1.5 * (w[:, :, None] * y).sum(dim=1))
    z = h @ p["head"].t()
    if own:
        b = xka.moe_balance_loss(logits, at, token_mask=mask)
        r = xka.token_logprobs(z, ids, 2)
        loss, lp, H, top = b.loss, r.logprobs, r.entropy, r.top_logprobs
    else:
        E = logits.shape[1]
        f = torch.bincount(at[mask].reshape(-1), minlength=E).to(x.dtype) / (k * mask.sum())
        loss = E * (f * prob[mask].mean(dim=0)).sum()
        ls = torch.log_softmax(z, dim=1)
        lp = torch.where(ids >= 0, ls.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0)
        H = -(ls.exp() * ls).sum(dim=1)
        top = torch.sort(ls, dim=1, descending=True, stable=True).values[:, :2]
    return -lp.sum() / mask.sum() + 0.01 * loss - 0.02 * H.mean() - 0.1 * top.mean()


def test_a_training_step_against_64_bits(cuda_device):
    """Gradients of every weight against torch's in 64 bits.  fp32 matrix products of 32 to 300 terms and the operators' own errors
    (at most some 2^-18 of what they add up) leave well under 2^-14 of a weight's gradient, in the norm."""
    p, x, ids, mask, k = model(cuda_device)
    got = {n: t.clone().requires_grad_() for n, t in p.items()}
    want = {n: t.double().requires_grad_() for n, t in p.items()}
    a, b = step(got, x, ids, mask, k, True), step(want, x.double(), ids, mask, k, False)
    assert abs(float(a.detach()) - float(b.detach())) <= 2.0 ** -16 * abs(float(b.detach()))
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        a.backward()
        b.backward()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    for n in p:
        g, w = got[n].grad.double(), want[n].grad
        assert float((g - w).norm()) <= 2.0 ** -14 * float(w.norm()), n


def test_gradients_that_nobody_asks_for(cuda_device):
    p, x, ids, mask, k = model(cuda_device)
    z = torch.randn(48, 300, device=cuda_device, requires_grad=True)
    r = xka.token_logprobs(z, ids, 2)
    assert not r.stats.requires_grad and not r.top_ids.requires_grad
    r.entropy.sum().backward()
    only = z.grad.clone()
    s = xkb.token_logprobs(z.detach(), ids)
    assert torch.equal(only, xkb.token_logprobs_backward(z.detach(), ids, s.stats, entropy=s.entropy, grad_entropy=torch.ones(48, device=cuda_device)))
    y = torch.randn(6, 2, 40, device=cuda_device, requires_grad=True)
    w = torch.rand(6, 2, device=cuda_device)
    xka.moe_sum_reduce(y, w).sum().backward()
    assert torch.equal(y.grad, w[:, :, None].expand(6, 2, 40))
    w.requires_grad_()
    xka.moe_sum_reduce(y.detach(), w).sum().backward()
    assert torch.allclose(w.grad, y.detach().sum(dim=2), atol=1e-4)
    xka.moe_sum_reduce(y).sum().backward()
    logits = torch.randn(6, 8, device=cuda_device, requires_grad=True)
    weights, at = xka.topk_softmax(logits, 2)
    assert weights.requires_grad and not at.requires_grad
    with torch.no_grad():
        assert not xka.topk_softmax(logits, 2)[0].requires_grad
    assert not xka.topk_softmax(logits.detach(), 2)[0].requires_grad
    plain = xkb.topk_softmax(logits.detach(), 2)
    assert torch.equal(weights, plain[0]) and torch.equal(at, plain[1])
    b = xka.moe_balance_loss(logits, at)
    assert b.loss.requires_grad and not b.counts.requires_grad


def functional_step(x, gate, head, ids, mask, k, y):
    """One step of the ops themselves, nothing read back."""
    logits, z = x @ gate.t(), x @ head.t()
    w, at = xkb.topk_softmax(logits, k)
    out = xkb.moe_sum_reduce(y, w)
    b = xkb.moe_balance_loss(logits, at, token_mask=mask)
    r = xkb.token_logprobs(z, ids, 4)
    g = torch.where(ids >= 0, -1.0, 0.0)
    gz = xkb.token_logprobs_backward(z, ids, r.stats, entropy=r.entropy, grad_logprobs=g, grad_entropy=0.1 * g)
    gy, gw = xkb.moe_sum_reduce_backward(out, y, w)
    gl = xkb.moe_router_backward(logits, at, grad_weights=gw, counts=b.counts, tokens=b.tokens, grad_loss=b.loss, token_mask=mask)
    return [out, *b, *r, gz, gy, gw, gl]


def inputs(dev, seed):
    p, x, ids, mask, k = model(dev)
    y = torch.randn(48, k, 32, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))
    return x + seed, p["gate"], p["head"], ids, mask, k, y


def test_captured_and_replayed(cuda_device):
    """Two captured steps, replayed on two streams at once, with inputs that change between replays."""
    args = [inputs(cuda_device, s) for s in (1, 2)]
    want = [functional_step(*a) for a in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(functional_step(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    fresh = inputs(cuda_device, 3)
    args[0][0].copy_(fresh[0])
    args[0][6].copy_(fresh[6])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], functional_step(*fresh)))


def test_the_differentiable_forms_refuse_capture(cuda_device):
    x = torch.randn(8, 16, device=cuda_device)
    leaf = x.clone().requires_grad_()
    ids = torch.zeros(8, dtype=torch.int64, device=cuda_device)
    xka.topk_softmax(x, 2)
    xka.token_logprobs(x, ids)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w, at = xka.topk_softmax(x, 2)            # nothing is recorded for a gradient
        for call in (lambda: xka.topk_softmax(leaf, 2), lambda: xka.token_logprobs(leaf, ids), lambda: xka.moe_balance_loss(leaf, at),
                     lambda: xka.moe_sum_reduce(leaf.view(8, 2, 8), w)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(at, xkb.topk_softmax(x, 2)[1])


def test_nor_does_their_backward_pass_run_in_one(cuda_device, monkeypatch):
    """(The answer of a capturing stream is put in its place: a captured backward pass is not started.)"""
    x, ids, y = torch.randn(8, 16, device=cuda_device), torch.zeros(8, dtype=torch.int64, device=cuda_device), torch.randn(8, 2, 4, device=cuda_device)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    w, at = xka.topk_softmax(leaf(x), 2)
    outs = [w, xka.token_logprobs(leaf(x), ids).logprobs, xka.moe_balance_loss(leaf(x), at).loss, xka.moe_sum_reduce(leaf(y), w.detach())]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for out in outs:
        with pytest.raises(RuntimeError, match="captured"):
            out.sum().backward()


def test_on_another_stream(cuda_device):
    """Inputs made on the stream that the calls run on, nothing waits for the default stream."""
    want = functional_step(*inputs(cuda_device, 4))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device=cuda_device)
        for _ in range(20):
            big = big @ big.t() * 1e-4
        got = functional_step(*inputs(cuda_device, 4))
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inputs_are_left_alone(cuda_device):
    a = inputs(cuda_device, 5)
    before = [t.clone() if isinstance(t, torch.Tensor) else t for t in a]
    functional_step(*a)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) if isinstance(p, torch.Tensor) else p == q for p, q in zip(a, before))
