"""What the logits of linear_cross_entropy lose where a sum is long: a large term first, and behind it terms of less than its last place."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import ops

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23


@pytest.fixture(autouse=True)
def no_wait_ran_out(cuda_device):
    yield
    ops.check_status(cuda_device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 8, 64, 77])
@pytest.mark.parametrize("H", [512, 1024, 4096])
def test_terms_below_the_last_place_of_few_rows(H, M, dtype, cuda_device):
    """z[7] = 1 + 0.75 ulp from every further 16 K.  A step of 16 K cuts off less than an ulp, and with few rows an accumulator takes
    128 K: the part with the 1 is off by less than 8 ulp.  The others hold multiples of 0.75 ulp alone, 6 ulp in all, and add up
    exactly."""
    x, w = torch.zeros(M, H, device=cuda_device), torch.zeros(1000, H, device=cuda_device)
    x[:, 0] = w[7, 0] = 1
    x[:, 16::16], w[7, 16::16] = 2.0 ** -12, 0.75 * 2.0 ** -11
    z = 1 + 0.75 * ULP * (H // 16 - 1)
    labels = torch.full((M,), 8, device=cuda_device)
    r = xkb.linear_cross_entropy(x.to(dtype), w.to(dtype), labels)
    assert float((r.stats[:, 0].double() - z).abs().max()) <= 8 * ULP
    # the sum of exponentials to 2^-20 as everywhere, and a rounding of l (6.9) and of lse (7.0)
    lse = z + math.log(1 + 999 * math.exp(-z))
    assert float((r.loss.double() - lse).abs().max()) <= 8 * ULP + 2.0 ** -19 + 8 * ULP


def test_sums_of_one_sign_do_not_drift(cuda_device):
    """Logits of positive terms, one row at a time: what is cut off adds up.  Of the eight steps of a part of 128 K each cuts off half an
    ulp on average, at most 2^-24 of the sum so far: 4.5 / 2 ulp of the part, and as much of the logit.  The parts' sums are rounded to
    nearest, 32 times, 0.3 ulp each with either sign: below 0.5 ulp in the mean over 16 rows.  So the mean is within 3 ulp."""
    H, V = 4096, 5003
    g = torch.Generator(device=cuda_device).manual_seed(3)
    w = (torch.rand(V, H, generator=g, device=cuda_device) * 0.02).to(torch.bfloat16)
    off = []
    for _ in range(16):
        x = torch.rand(1, H, generator=g, device=cuda_device).to(torch.bfloat16)
        z = (x.double() @ w.double().t())[0]
        r = xkb.linear_cross_entropy(x, w, z.argmax()[None])
        off.append(float((r.stats[0, 0].double() - z.max()) / z.max()))
    assert abs(sum(off)) / len(off) <= 3 * ULP, off


@pytest.mark.parametrize("M", [129, 300, 1000])
@pytest.mark.parametrize("H", [512, 2048, 4096])
def test_terms_below_the_last_place_of_many_rows(H, M, cuda_device):
    """The same with parts of 512 K: 32 steps of less than an ulp; the other parts hold 24 ulp each, and add up exactly."""
    x, w = torch.zeros(M, H, device=cuda_device), torch.zeros(1000, H, device=cuda_device)
    x[:, 0] = w[7, 0] = 1
    x[:, 16::16], w[7, 16::16] = 2.0 ** -12, 0.75 * 2.0 ** -11
    z = 1 + 0.75 * ULP * (H // 16 - 1)
    r = xkb.linear_cross_entropy(x.to(torch.bfloat16), w.to(torch.bfloat16), torch.full((M,), 8, device=cuda_device))
    assert float((r.stats[:, 0].double() - z).abs().max()) <= 32 * ULP
