"""moe_balance_loss and moe_router_backward against 64 bits: expert counts around the pieces of a row, dropped slots, masked
tokens, dead and NaN rows; the gradient against the formula and against differences."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from tests import loss_util as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def case(M, E, k, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(M * 7 + E * 3 + k + seed)
    x = (torch.randn(M, E, generator=g, device=dev) * 1.5).to(dtype)
    w, ids = xkb.topk_softmax(x, k) if M else (None, torch.zeros(0, k, dtype=torch.int32, device=dev))
    return x, ids, torch.randn(M, k, generator=g, device=dev), torch.rand(M, generator=g, device=dev) < 0.7


def check_loss(x, ids, mask=None):
    got = xkb.moe_balance_loss(x, ids, token_mask=mask)
    loss, counts, mean, T = ref.balance(x, ids, mask)
    assert got.loss.shape == () and got.tokens.shape == () and int(got.tokens) == T
    assert got.counts.dtype == torch.int32 and torch.equal(got.counts.long(), counts)
    # exponentials and divisions; a warp's rows in turn (at least one warp in eight of 296 blocks), the joins
    rel = 2.0 ** -20 + (x.shape[0] / 2368 + 600) * ref.U24
    ref.assert_near(got.mean_probs, mean, rel * mean.nan_to_num(0).abs(), "mean_probs")
    ref.assert_near(got.loss, loss, 2 * rel * loss.nan_to_num(0).abs(), "loss")
    return got


def check_grad(x, ids, g_w, renorm, counts=None, tokens=None, g_loss=None, mask=None):
    got = xkb.moe_router_backward(x, ids, grad_weights=g_w, renormalize=renorm, counts=counts, tokens=tokens, grad_loss=g_loss,
                                  token_mask=mask)
    want, err = ref.router_grad(x, ids, g_w, renorm, counts, tokens, 1.0 if g_loss is None else g_loss, mask)
    assert got.dtype == x.dtype and got.is_contiguous()
    ref.assert_near(got, want, err, "gradient")
    return got


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (4, 4), (8, 2), (31, 3), (32, 8), (33, 8), (48, 8), (60, 6), (64, 40), (96, 33),
                                 (127, 2), (256, 8), (257, 8), (384, 8), (512, 10), (1000, 8), (1024, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_experts(E, k, dtype, cuda_device):
    for M in (1, 19, 333):
        x, ids, g_w, mask = case(M, E, k, dtype, cuda_device)
        check_loss(x, ids)
        r = check_loss(x, ids, mask)
        for renorm in (True, False):
            check_grad(x, ids, g_w, renorm)
            check_grad(x, ids, g_w, renorm, r.counts, r.tokens, 0.3, mask)
        check_grad(x, ids, None, True, r.counts)
        check_grad(x, ids, None, True, r.counts, r.tokens, torch.tensor(-2.0, device=cuda_device), mask)


@pytest.mark.parametrize("M", [0, 1, 7, 8, 9, 2367, 2368, 2369, 40001])
def test_tokens(M, cuda_device):
    x, ids, g_w, mask = case(M, 64, 4, torch.bfloat16, cuda_device)
    r = check_loss(x, ids)
    check_loss(x, ids, mask)
    check_grad(x, ids, g_w, True, r.counts, r.tokens, 0.01)


def test_an_even_routing_has_loss_one(cuda_device):
    x = torch.zeros(64, 16, device=cuda_device)
    ids = (torch.arange(64 * 2, device=cuda_device, dtype=torch.int32) % 16).reshape(64, 2)
    assert abs(float(xkb.moe_balance_loss(x, ids).loss) - 1.0) < 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropped_slots_and_masked_tokens(dtype, cuda_device):
    x, ids, g_w, mask = case(500, 48, 6, dtype, cuda_device)
    ids = torch.where(torch.rand(500, 6, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(9)) < 0.3, -1, ids)
    ids[3] = -1                                    # a token without an expert
    ids[4, 0], ids[5, 1], ids[6, 2] = 48, 2 ** 31 - 1, -2 ** 31
    g_w[7, ids[7] < 0] = math.nan                  # of a dropped slot: not looked at
    x[8] = -math.inf                               # dead
    x[9] = torch.finfo(dtype).min                  # even
    x[10, 5:] = -math.inf
    r = check_loss(x, ids, mask)
    for renorm in (True, False):
        check_grad(x, ids, g_w, renorm, r.counts, r.tokens, 1.0, mask)
    check_loss(x, ids.long(), mask.to(torch.uint8))
    none = torch.zeros_like(mask)
    r = check_loss(x, ids, none)
    assert float(r.loss) == 0.0 and int(r.tokens) == 0
    assert not bool(check_grad(x, ids, None, True, r.counts, r.tokens, 1.0, none).any())


def test_wide_ids_are_dropped_slots_too(cuda_device):
    """int64 ids that no int32 holds do not wrap around to an expert."""
    x, ids, g_w, _ = case(40, 16, 4, torch.float32, cuda_device)
    wide = ids.long()
    wide[::3, 0], wide[1::3, 1] = 2 ** 32 + 3, -(2 ** 33)
    check_loss(x, wide)
    check_grad(x, wide, g_w, True)


def test_padding_may_hold_anything(cuda_device):
    """Rows behind the mask, and rows that no gradient comes back to, are not looked at."""
    x, ids, g_w, mask = case(200, 64, 4, torch.float32, cuda_device)
    want, clean = xkb.moe_balance_loss(x, ids, token_mask=mask), x.clone()
    g_w[~mask] = 0.0
    x[~mask] = math.nan
    got = xkb.moe_balance_loss(x, ids, token_mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for kw in (dict(grad_weights=g_w), dict(counts=got.counts, tokens=got.tokens), dict(grad_weights=g_w, counts=got.counts, tokens=got.tokens)):
        a, b = (xkb.moe_router_backward(z, ids, token_mask=mask, **kw) for z in (x, clean))
        assert torch.equal(a[mask], b[mask]) and not bool(a[~mask].any())


def test_nan_shows(cuda_device):
    x, ids, g_w, _ = case(50, 40, 4, torch.bfloat16, cuda_device)
    x[3, 7], x[4, 8] = math.nan, math.inf
    r = xkb.moe_balance_loss(x, ids)
    assert bool(r.loss.isnan()) and bool(r.mean_probs.isnan().all())
    got = xkb.moe_router_backward(x, ids, grad_weights=g_w)
    bad = got.isnan().all(dim=1)
    assert bool(bad[3:5].all()) and int(bad.sum()) == 2


@pytest.mark.parametrize("renorm", [True, False])
def test_an_expert_named_twice(renorm, cuda_device):
    x, ids, g_w, _ = case(64, 50, 5, torch.float32, cuda_device)
    ids[:, 1] = ids[:, 0]
    ids[::2, 3] = ids[::2, 0]
    check_grad(x, ids, g_w, renorm)
    x, ids, g_w, _ = case(64, 50, 40, torch.float32, cuda_device)
    ids[:, 35:] = ids[:, :1]
    check_grad(x, ids, g_w, renorm)


@pytest.mark.parametrize("E,k", [(65, 8), (128, 8), (128, 9), (97, 16), (128, 17), (130, 16), (256, 16), (255, 17), (258, 16), (512, 16), (512, 17),
                                 (513, 16)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_warps(E, k, dtype, cuda_device):
    """The layouts of a row over 8, 16 and 32 lanes, with several rounds of rows and experts named twice."""
    for M in (3, 20011 if E <= 256 else 12007):
        x, ids, g_w, mask = case(M, E, k, dtype, cuda_device)
        ids[::3, 1] = ids[::3, 0]
        ids[1::5, k - 1] = ids[1::5, 2]
        r = check_loss(x, ids, mask)
        check_grad(x, ids, g_w, True, r.counts, r.tokens, 0.3, mask)
        check_grad(x, ids, g_w, False)


def test_sharp_rows(cuda_device):
    """Probabilities down to 0, selected ones among them."""
    x, ids, g_w, _ = case(64, 64, 8, torch.float32, cuda_device)
    x *= torch.logspace(-3, 3, 64, device=cuda_device)[:, None]
    w, ids = xkb.topk_softmax(x, 8)
    check_grad(x, ids, g_w, True)
    check_grad(x, ids, g_w, False)
    far = torch.sort(x, dim=1).indices[:, :8].to(torch.int32)      # the least likely: their sum may be 0
    got = xkb.moe_router_backward(x, far, grad_weights=g_w, renormalize=False)
    want, err = ref.router_grad(x, far, g_w, False)
    ref.assert_near(got, want, err)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned(dtype, cuda_device):
    x, ids, g_w, mask = case(40, 64, 4, dtype, cuda_device)
    flat = torch.empty(40 * 64 + 1, dtype=dtype, device=cuda_device)
    odd = flat[1:].view(40, 64)
    odd.copy_(x)
    for y in (odd, x.t().contiguous().t(), torch.cat([x, x], dim=1)[:, :64]):
        a, b = xkb.moe_balance_loss(y, ids), xkb.moe_balance_loss(x, ids)
        assert torch.equal(a.counts, b.counts) and torch.allclose(a.mean_probs, b.mean_probs, rtol=1e-5)
        check_grad(y, ids, g_w, True, a.counts, a.tokens)
    wide = torch.randn(40, 8, device=cuda_device)
    check_grad(x, ids.t().contiguous().t(), wide[:, ::2], True, torch.stack([b.counts, b.counts], 1)[:, 0].long(), b.tokens[None])
    check_loss(x, ids, torch.stack([mask, mask], 1)[:, 0])


def test_counts_of_several_ranks(cuda_device):
    """Summed counts and tokens give the gradient of the whole batch's loss."""
    x, ids, _, mask = case(300, 32, 4, torch.float32, cuda_device)
    whole = xkb.moe_balance_loss(x, ids, token_mask=mask)
    parts = [xkb.moe_balance_loss(x[s], ids[s], token_mask=mask[s]) for s in (slice(0, 100), slice(100, 300))]
    counts, tokens = sum(p.counts for p in parts), sum(p.tokens for p in parts)
    assert torch.equal(counts, whole.counts) and int(tokens) == int(whole.tokens)
    got = [xkb.moe_router_backward(x[s], ids[s], counts=counts, tokens=tokens, token_mask=mask[s]) for s in (slice(0, 100), slice(100, 300))]
    assert torch.equal(torch.cat(got), xkb.moe_router_backward(x, ids, counts=whole.counts, tokens=whole.tokens, token_mask=mask))


def test_against_differences(cuda_device):
    x, ids, g_w, mask = case(30, 40, 5, torch.float32, cuda_device)
    r = xkb.moe_balance_loss(x, ids, token_mask=mask)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    for renorm in (True, False):
        got = check_grad(x, ids, g_w, renorm, r.counts, r.tokens, 0.7, mask).double()

        def f(z):
            p = torch.softmax(z, dim=1)
            w = p.gather(1, ids.long())
            if renorm:
                w = w / w.sum(dim=1, keepdim=True)
            return (w * g_w.double()).sum() + 0.7 * ref.balance(z, ids, mask)[0]

        _, err = ref.router_grad(x, ids, g_w, renorm, r.counts, r.tokens, 0.7, mask)
        for _ in range(4):
            v, h = torch.randn(30, 40, generator=g, device=cuda_device, dtype=torch.float64), 1e-5
            want = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
            bound = ((err + ref.U24 * got.abs() + 1e-9) * v.abs()).sum()
            assert abs(float((got * v).sum() - want)) <= float(bound)


def test_same_bits(cuda_device):
    x, ids, g_w, mask = case(30001, 100, 8, torch.bfloat16, cuda_device)
    a, b = (xkb.moe_balance_loss(x, ids, token_mask=mask) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a, b = (xkb.moe_router_backward(x, ids, grad_weights=g_w, counts=a.counts, tokens=a.tokens, token_mask=mask) for _ in range(2))
    assert torch.equal(a, b)


def test_refusals(cuda_device):
    x, ids, g_w, mask = case(8, 16, 2, torch.float32, cuda_device)
    r = xkb.moe_balance_loss(x, ids)
    loss, grad = xkb.moe_balance_loss, xkb.moe_router_backward
    from xkernels_b200._lib import XkbError

    for call, error in ((lambda: loss(x.cpu(), ids), RuntimeError), (lambda: loss(x, ids[:4]), ValueError), (lambda: loss(x, None), TypeError),
                        (lambda: loss(x, ids.float()), TypeError), (lambda: loss(x.double(), ids), TypeError), (lambda: loss(x[0], ids), ValueError),
                        (lambda: loss(x, ids, token_mask=mask[:3]), ValueError), (lambda: loss(x, ids, token_mask=mask.float()), TypeError),
                        (lambda: loss(torch.zeros(8, 1025, device=cuda_device), ids), XkbError), (lambda: loss(x[:, :0], ids), ValueError),
                        (lambda: grad(x, ids), ValueError), (lambda: grad(x, ids, grad_weights=g_w[:, :1]), ValueError),
                        (lambda: grad(x, ids, grad_weights=g_w, grad_loss=1.0), ValueError), (lambda: grad(x, None, grad_weights=g_w), TypeError),
                        (lambda: grad(x, ids, counts=r.counts[:3]), ValueError), (lambda: grad(x, ids, counts=r.counts.cpu()), RuntimeError),
                        (lambda: grad(torch.zeros(8, 1025, device=cuda_device), ids, grad_weights=g_w), XkbError)):
        with pytest.raises(error):
            call()
