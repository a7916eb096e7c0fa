"""moe_router_backward for choices that are not the row's most likely experts: renormalised weights depend on the chosen logits
alone, however far these lie below the row's largest one."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from tests import loss_util as ref
from xkernels_b200 import autograd as xka

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def renormalised_grad(x, ids, g_w, counts=None, tokens=None, g_loss=1.0):
    """(gradient, the magnitude that its errors are relative to) in 64 bits.  The weights are a softmax over the chosen logits, formed
    from differences to the largest of them: no sum is 0 where a chosen logit is live."""
    E, k = x.shape[1], ids.shape[1]
    valid = (ids >= 0) & (ids < E)
    at = ids.long().clamp(0, E - 1)
    z = torch.where(valid, x.double().gather(1, at), -math.inf)
    w = ref.softmax_or_zero(z)
    g = torch.where(valid, g_w.double(), 0.0)
    part = w * (g - (w * g).sum(dim=1, keepdim=True))
    d = torch.zeros_like(x, dtype=torch.float64).scatter_add_(1, at, part)
    # An exponential of y = difference x log2(e) errs by 2^-21 and by the rounding of y, 2^-24 of |y|; the difference is to the largest chosen
    # logit (-ln w at most), or to the row's where the chosen ones still have 2^-20 of its probability (14 more).  As in loss_util: four
    # times that for sums, quotients and products.
    depth = torch.where(w > 0, -w.clamp(min=1e-300).log(), 0.0) + 14
    size = w * (g.abs() + (w * g.abs()).sum(dim=1, keepdim=True)) * (2.0 ** -19 + depth * 2.0 ** -23)
    err = torch.zeros_like(d).scatter_add_(1, at, size)
    # an exponential below 2^-126 is flushed to 0, which is 2^-106 of a weight where the chosen ones have 2^-20 of the row
    err = err.scatter_add_(1, at, 2.0 ** -105 * (g.abs() + g.abs().sum(dim=1, keepdim=True)))
    if counts is not None:
        more, more_err = ref.router_grad(x, ids, None, True, counts, tokens, g_loss)
        d, err = d + more, err + more_err
    return d, err


def case(M, E, k, dtype, dev, depth, seed=0):
    """Rows whose ids are the least likely experts, ``depth`` nats and more below the row's largest logit."""
    g = torch.Generator(device=dev).manual_seed(M * 7 + E * 3 + k + seed)
    x = torch.randn(M, E, generator=g, device=dev)
    ids = torch.argsort(torch.rand(M, E, generator=g, device=dev), dim=1)[:, :k].to(torch.int32).contiguous()
    x.scatter_add_(1, ids.long(), torch.full((M, k), -float(depth), device=dev))
    return x.to(dtype), ids, torch.randn(M, k, generator=g, device=dev)


def check(x, ids, g_w, balance=False):
    kw = {}
    if balance:
        r = xkb.moe_balance_loss(x, ids)
        kw = dict(counts=r.counts, tokens=r.tokens)
    got = xkb.moe_router_backward(x, ids, grad_weights=g_w, renormalize=True, grad_loss=0.3 if balance else None, **kw)
    want, err = renormalised_grad(x, ids, g_w, g_loss=0.3, **kw)
    ref.assert_near(got, want, err, "gradient")
    return got


def test_the_form_agrees_with_autograd():
    x, ids, g_w = case(20, 30, 4, torch.float32, "cpu", 3.0)
    leaf = x.double().requires_grad_()
    w = torch.softmax(leaf, dim=1).gather(1, ids.long())
    ((w / w.sum(dim=1, keepdim=True)) * g_w.double()).sum().backward()
    assert torch.allclose(renormalised_grad(x, ids, g_w)[0], leaf.grad, rtol=1e-12, atol=1e-15)



# every layout of a row: 8, 16 and 32 lanes, one to 32 experts a lane, and more slots than lanes
SHAPES = [(8, 3), (16, 4), (31, 3), (48, 8), (60, 6), (64, 40), (128, 8), (128, 9), (255, 8), (256, 8), (256, 33), (384, 8), (500, 16), (512, 10),
          (1000, 8), (1024, 64)]


@pytest.mark.parametrize("E,k", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_below_the_row(E, k, dtype, cuda_device):
    """Depths around the smallest exponential (87 nats), where a sum over the chosen ones is 0 or its inverse near 2^126, and beyond."""
    for depth in (13.0, 14.0, 20.0, 80.0, 84.0, 86.0, 87.0, 88.0, 90.0, 104.0, 1000.0):
        x, ids, g_w = case(37, E, k, dtype, cuda_device, depth)
        got = check(x, ids, g_w * 100)
        assert bool((got != 0).any(dim=1).all())
        check(x, ids, g_w, balance=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_least_likely_of_sharp_rows(dtype, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(64, 64, generator=g, device=cuda_device) * torch.logspace(-3, 3, 64, device=cuda_device)[:, None]
    x = x.to(dtype)
    g_w = torch.randn(64, 8, generator=g, device=cuda_device)
    far = torch.sort(x.float(), dim=1, stable=True).indices[:, :8].to(torch.int32)
    check(x, far, g_w)
    check(x, far, g_w, balance=True)
    far[::3, 0] = -1                           # dropped slots among them
    far[1::3, 2] = far[1::3, 1]                # and an expert named twice
    check(x, far, g_w)


def test_masks_among_the_chosen(cuda_device):
    x, ids, g_w = case(12, 40, 4, torch.float32, cuda_device, 200.0)
    at = ids.long()
    x[0].scatter_(0, at[0], -math.inf)         # no chosen expert is live: no gradient
    x[1, at[1, 0]] = -math.inf                 # one of them is not
    x[2].scatter_(0, at[2], torch.finfo(torch.float32).min)    # a mask of the lowest value: even weights
    x[3] = -math.inf
    ids[4] = -1
    x[5] -= 3e6                                # far from zero, whole steps of 1/4
    x[6, at[6]] = 1e30
    got = check(x, ids, g_w)
    assert not bool(got[[0, 3, 4]].any()) and bool((got[2] != 0).any())


def test_a_row_does_not_depend_on_its_neighbours(cuda_device):
    """Rows far below and ordinary ones share a warp: each has the bits that it has alone."""
    a, ids, g_w = case(64, 64, 6, torch.float32, cuda_device, 95.0)
    b, _, _ = case(64, 64, 6, torch.float32, cuda_device, 0.5)
    x = torch.where((torch.arange(64, device=cuda_device) % 3 == 0)[:, None], a, b)
    got = xkb.moe_router_backward(x, ids, grad_weights=g_w)
    rows = [xkb.moe_router_backward(x[i:i + 1], ids[i:i + 1], grad_weights=g_w[i:i + 1]) for i in range(64)]
    assert torch.equal(got, torch.cat(rows))


def test_against_differences(cuda_device):
    """sum of dx v against (f(x + h v) - f(x - h v)) / 2h in 64 bits, whose error is about h^2 + 2^-52 / h."""
    x, ids, g_w = case(30, 40, 5, torch.float32, cuda_device, 95.0)
    got = xkb.moe_router_backward(x, ids, grad_weights=g_w).double()
    _, err = renormalised_grad(x, ids, g_w)
    g = torch.Generator(device=cuda_device).manual_seed(2)

    def f(z):
        return (torch.softmax(z.gather(1, ids.long()), dim=1) * g_w.double()).sum()

    for _ in range(4):
        v, h = torch.randn(30, 40, generator=g, device=cuda_device, dtype=torch.float64), 1e-5
        want = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
        assert abs(float((got * v).sum() - want)) <= float(((err + ref.U24 * got.abs() + 1e-9) * v.abs()).sum())


# ---- slots that are dropped behind the router -------------------------------------------------------------------
def routing64(leaf, ids):
    p = torch.softmax(leaf, dim=1).gather(1, ids.long())
    return p / p.sum(dim=1, keepdim=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_slots_dropped_behind_the_router(dtype, cuda_device):
    """topk_softmax, then a slot is dropped (an expert's capacity): the weights were formed over all top_k slots, so the gradient takes the
    ids that topk_softmax gave and 0 for what was dropped.  The balance loss counts the kept slots alone.  Against autograd
    of that composition in 64 bits."""
    M, E, k = 300, 48, 6
    g = torch.Generator(device=cuda_device).manual_seed(8)
    x = (torch.randn(M, E, generator=g, device=cuda_device) * 1.5).to(dtype)
    keep = torch.rand(M, k, generator=g, device=cuda_device) < 0.7
    keep[0] = False
    g_w = torch.randn(M, k, generator=g, device=cuda_device)
    _, ids = xkb.topk_softmax(x, k)
    kept_ids = torch.where(keep, ids, -1)
    r = xkb.moe_balance_loss(x, kept_ids)
    got = xkb.moe_router_backward(x, ids, grad_weights=torch.where(keep, g_w, 0.0), counts=r.counts, tokens=r.tokens, grad_loss=0.3)

    leaf = x.double().requires_grad_()
    loss = (routing64(leaf, ids) * keep * g_w.double()).sum()
    (loss + 0.3 * E * (r.counts.double() / (k * M) * torch.softmax(leaf, dim=1).mean(dim=0)).sum()).backward()
    _, err = ref.router_grad(x, ids, torch.where(keep, g_w, 0.0), True, r.counts, r.tokens, 0.3)
    ref.assert_near(got, leaf.grad, err, "gradient")


def test_slots_dropped_through_autograd(cuda_device):
    """The differentiable router keeps its own ids: dropping is a matter of what becomes of the weights."""
    g = torch.Generator(device=cuda_device).manual_seed(9)
    x = torch.randn(200, 32, generator=g, device=cuda_device)
    keep = torch.rand(200, 4, generator=g, device=cuda_device) < 0.7
    g_w = torch.randn(200, 4, generator=g, device=cuda_device)
    own, plain = x.clone().requires_grad_(), x.double().requires_grad_()
    w, ids = xka.topk_softmax(own, 4)
    (w * keep * g_w).sum().backward()
    (routing64(plain, ids) * keep * g_w.double()).sum().backward()
    _, err = ref.router_grad(x, ids, torch.where(keep, g_w, 0.0), True)
    ref.assert_near(own.grad, plain.grad, err + 2 ** -23 * plain.grad.abs())
    w, ids = xka.topk_softmax(own, 4)
    ids[~keep] = -1                            # the ids that the gradient needs: torch refuses
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()


def test_weights_of_the_kept_slots(cuda_device):
    """Ids outside [0, E) mean weights that were formed over the kept slots: p_j by the sum of the kept p."""
    g = torch.Generator(device=cuda_device).manual_seed(10)
    x = torch.randn(200, 32, generator=g, device=cuda_device)
    _, ids = xkb.topk_softmax(x, 4)
    keep = torch.rand(200, 4, generator=g, device=cuda_device) < 0.7
    keep[:, 0] = True
    g_w = torch.randn(200, 4, generator=g, device=cuda_device)
    kept_ids = torch.where(keep, ids, 32)
    leaf = x.double().requires_grad_()
    p = torch.softmax(leaf, dim=1).gather(1, ids.long()) * keep
    (p / p.sum(dim=1, keepdim=True) * g_w.double()).sum().backward()
    _, err = ref.router_grad(x, kept_ids, g_w, True)
    ref.assert_near(xkb.moe_router_backward(x, kept_ids, grad_weights=g_w), leaf.grad, err)


@pytest.mark.parametrize("dtype", DTYPES)
def test_both_losses_on_the_same_logits(dtype, cuda_device):
    """Through the differentiable forms the two gradients are results of their own, each rounded, and torch rounds their sum."""
    M, E, k = 333, 60, 6
    g = torch.Generator(device=cuda_device).manual_seed(12)
    x = (torch.randn(M, E, generator=g, device=cuda_device) * 1.5).to(dtype)
    g_w = torch.randn(M, k, generator=g, device=cuda_device)
    mask = torch.rand(M, generator=g, device=cuda_device) < 0.8
    leaf = x.clone().requires_grad_()
    w, ids = xka.topk_softmax(leaf, k)
    b = xka.moe_balance_loss(leaf, ids, mask)
    ((w * g_w).sum() + 300.0 * b.loss).backward()
    parts = [ref.router_grad(x, ids, g_w, True), ref.router_grad(x, ids, None, True, b.counts, b.tokens, 300.0, mask)]
    err = sum(e + ref.half_step(dtype) * (d.abs() + e) + ref.TINY[dtype] for d, e in parts)
    ref.assert_near(leaf.grad, parts[0][0] + parts[1][0], err + ref.half_step(dtype) * err)
