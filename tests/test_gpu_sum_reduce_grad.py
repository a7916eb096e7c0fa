"""moe_sum_reduce_backward against 64 bits: columns around a vector, a warp and a block, few and many slots and tokens."""

import pytest
import torch

import xkernels_b200 as xkb
from tests import loss_util as ref

pytestmark = pytest.mark.gpu


def check(go, y, w, f=1.0, **need):
    gy, gw = xkb.moe_sum_reduce_backward(go, y, w, f, **need)
    M, k, H = y.shape
    wd = torch.ones(M, k, dtype=torch.float64, device=y.device) if w is None else w.double()
    if need.get("need_grad_y", True):
        want = f * wd[:, :, None] * go.double()[:, None, :]
        assert gy.dtype == y.dtype and gy.is_contiguous()
        ref.assert_near(gy, want, 3 * ref.U24 * want.abs(), "grad_y")     # f, f w and the product
    else:
        assert gy is None
    if w is not None and need.get("need_grad_w", True):
        term = f * go.double()[:, None, :] * y.double()
        assert gw.dtype == w.dtype
        # at most H / 32 terms one after the other, the joins
        ref.assert_near(gw, term.sum(dim=2), (H / 32 + 48) * ref.U24 * term.abs().sum(dim=2), "grad_w")
    else:
        assert gw is None
    return gy, gw


def case(M, k, H, dtype, dev, w_dtype=torch.float32):
    g = torch.Generator(device=dev).manual_seed(M + 100 * k + H)
    return (torch.randn(M, H, generator=g, device=dev).to(dtype), torch.randn(M, k, H, generator=g, device=dev).to(dtype),
            torch.randn(M, k, generator=g, device=dev).to(w_dtype))


@pytest.mark.parametrize("H", [1, 4, 7, 8, 12, 64, 136, 256, 1000, 2048, 2056, 4100, 7168])
@pytest.mark.parametrize("k", [1, 2, 3, 6, 8, 9, 17])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sizes(H, k, dtype, cuda_device):
    for M in (1, 5, 160):
        check(*case(M, k, H, dtype, cuda_device), 2.5)
    check(*case(3, k, H, dtype, cuda_device, torch.bfloat16))


@pytest.mark.parametrize("M", [147, 148, 296, 297, 593, 1184, 20011])
@pytest.mark.parametrize("H", [8, 32, 64, 72, 512])
def test_many_narrow_tokens(M, H, cuda_device):
    for k in (1, 3, 8):
        check(*case(M, k, H, torch.bfloat16, cuda_device))
        check(*case(M, k, H, torch.float32, cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parts(dtype, cuda_device):
    go, y, w = case(40, 6, 264, dtype, cuda_device)
    both = check(go, y, w)
    assert torch.equal(check(go, y, w, need_grad_w=False)[0], both[0])
    assert torch.equal(check(go, y, w, need_grad_y=False)[1], both[1])
    check(go, y, None, 0.5)
    check(go, y, w, need_grad_y=False, need_grad_w=False)
    check(go, y, w.half().float())
    gy, gw = xkb.moe_sum_reduce_backward(go, y, w.half())
    assert gw.dtype == torch.float16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dtype, cuda_device):
    go, y, w = case(12, 4, 64, dtype, cuda_device)
    want = check(go, y, w)
    odd = torch.empty(12 * 4 * 64 + 1, dtype=dtype, device=cuda_device)[1:].view(12, 4, 64)
    odd.copy_(y)
    got = check(go, odd, w)
    assert torch.equal(got[0], want[0])
    check(go, y.transpose(0, 1).contiguous().transpose(0, 1), w)
    check(go[:1].expand(12, 64), y, w.t().contiguous().t())       # the gradient of a sum
    check(go.t().contiguous().t(), y, w)


def shifted(t, by):
    """The same values, `by` elements behind a 16-byte boundary."""
    out = torch.full((t.numel() + by + 8,), float("nan"), dtype=t.dtype, device=t.device)[by:by + t.numel()].view(t.shape)
    return out.copy_(t)


@pytest.mark.parametrize("H", [1, 2, 3, 5, 7, 9, 15, 17, 33, 255, 257, 333, 1001, 2047, 2049, 4095, 4098, 4100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_start_anywhere(H, dtype, cuda_device):
    for M, k in ((1, 1), (1, 2), (2, 5), (7, 3), (151, 2), (301, 3), (299, 8), (300, 10)):
        c = case(M, k, H, dtype, cuda_device)
        check(*c, 2.5)
    go, y, w = case(300, 6, H, dtype, cuda_device)
    for by_go, by_y in ((1, 0), (0, 1), (3, 2), (5, 7)):
        go1, y1 = shifted(go, by_go), shifted(y, by_y)
        check(go1, y1, w)
        check(go1, y1, w, need_grad_y=False)
        check(go1, y1, w, need_grad_w=False)


@pytest.mark.parametrize("H", [3, 17, 333, 1000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_keep_to_themselves(H, dtype, cuda_device):
    go, y, w = case(320, 6, H, dtype, cuda_device)
    want = xkb.moe_sum_reduce_backward(go, y, w)
    go1, y1 = go.clone(), y.clone()
    y1[1::5, 2], y1[3::7, 5], go1[::6] = float("nan"), float("inf"), float("nan")
    gy, gw = xkb.moe_sum_reduce_backward(go1, y1, w)
    live_y = torch.ones(320, 6, dtype=torch.bool, device=cuda_device)
    live_y[::6] = False
    live_w = live_y.clone()
    live_w[1::5, 2] = live_w[3::7, 5] = False
    assert torch.equal(gy[live_y], want[0][live_y]) and torch.equal(gw[live_w], want[1][live_w])
    assert bool(gy[::6].isnan().all()) and not bool(gw[~live_w].isfinite().any())


def test_nothing_to_do(cuda_device):
    for M, k, H in ((0, 2, 8), (3, 0, 8), (3, 2, 0)):
        gy, gw = xkb.moe_sum_reduce_backward(torch.ones(M, H, device=cuda_device), torch.ones(M, k, H, device=cuda_device),
                                             torch.ones(M, k, device=cuda_device))
        assert gy.shape == (M, k, H) and gw.shape == (M, k) and not bool(gw.any())


def test_rows_behind_two_to_the_31(cuda_device):
    M, k, H = 40000, 8, 7168
    y = torch.zeros(M, k, H, dtype=torch.bfloat16, device=cuda_device)
    go = torch.zeros(M, H, dtype=torch.bfloat16, device=cuda_device)
    a, b, w = case(2, k, H, torch.bfloat16, cuda_device)
    go[-2:], y[-2:] = a, b
    gy, gw = xkb.moe_sum_reduce_backward(go, y, torch.cat([torch.ones(M - 2, k, device=cuda_device), w]))
    want = xkb.moe_sum_reduce_backward(a, b, w)
    assert torch.equal(gy[-2:], want[0]) and torch.allclose(gw[-2:], want[1], rtol=1e-4, atol=1e-3) and not bool(gw[:-2].any())


def test_same_bits(cuda_device):
    c = case(700, 8, 1000, torch.bfloat16, cuda_device)
    a, b = (xkb.moe_sum_reduce_backward(*c) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals(cuda_device):
    go, y, w = case(4, 2, 16, torch.float32, cuda_device)
    f = xkb.moe_sum_reduce_backward
    for call, error in ((lambda: f(go.cpu(), y, w), RuntimeError), (lambda: f(go, y[0], w), ValueError), (lambda: f(go[:3], y, w), ValueError),
                        (lambda: f(go, y, w[:, :1]), ValueError), (lambda: f(go, y.half(), w), TypeError)):
        with pytest.raises(error):
            call()
