"""Gradients of tokens that the head is sure of: 1 - p is small, and d = (p - 1) a is no better than the logits that are multiplied once
more."""

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import ops

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23


# An accumulator cuts half an ulp off the sum for each 16 K on average, and off each of the 16 products what lies two bits below its last
# place or lower (products of fp16 numbers have 22 bits), an eighth of an ulp on average: 2.5 ulp of the sum so far.  Of z, in parts of
# 128 K (up to 128 rows) 4.5 * 2.5 ulp, in parts of 512 K 16.5 * 2.5.  (In one part of 4096 K 128 * 1.2 are seen.)
SHORT, LONG = 4.5 * 2.5, 16.5 * 2.5


@pytest.mark.parametrize("M,V,ulps", [(10, 64, SHORT), (100, 64, SHORT), (300, 64, LONG), (1000, 64, LONG), (100, 8192, SHORT), (300, 8192, LONG),
                                      (1000, 8192, LONG)])
@pytest.mark.parametrize("H", [1024, 4096])
def test_the_labels_gradient(H, M, V, ulps, cuda_device):
    """A column that is 1 in the label's weights and 0 elsewhere reads d of the label.  z = 16 or so, of positive terms, the others half of
    it or a fifth: 1 - p = 0.02.  The roundings of d and of the result are 2^-11 of 1 - p each, of either sign: in the mean over the rows
    three of their standard deviations."""
    dt = torch.float16
    g = torch.Generator(device=cuda_device).manual_seed(H + M)
    w0 = (0.5 + torch.rand(H, generator=g, device=cuda_device)) / 64
    w = (w0 * (torch.linspace(0.45, 0.55, V, device=cuda_device) - (0.3 if V > 64 else 0))[:, None]).to(dt)
    w[0] = w0.to(dt)
    x = ((0.5 + torch.rand(M, H, generator=g, device=cuda_device)) * 64 * 16 / H).to(dt)
    w, x = (torch.cat([t, torch.zeros(len(t), 8, dtype=dt, device=cuda_device)], dim=1) for t in (w, x))
    w[0, H] = 1
    z = x.double() @ w.double().t()
    m = z.amax(dim=1, keepdim=True)
    l = torch.logsumexp(z - m, dim=1, keepdim=True)
    p = (z[:, 0:1] - m - l).exp()[:, 0]
    assert 14 < float(z[:, 0].min()) and float(z[:, 0].max()) < 18 and 0.001 < float((1 - p).min())
    labels, stats = torch.zeros(M, dtype=torch.int64, device=cuda_device), torch.cat([m, l], dim=1).float()
    gx, _ = xkb.linear_cross_entropy_backward(x, w, labels, stats, grad_loss=torch.ones(M, device=cuda_device))
    ops.check_status(cuda_device)
    off = (gx[:, H].double() - (p - 1)) / (p * z[:, 0])          # d p = p d z
    noise = 2 * float(((1 - p) / (p * z[:, 0])).mean()) * 2.0 ** -11 / 3 ** 0.5 / M ** 0.5
    # the statistics given are rounded to fp32 once, and exponents of p: an ulp
    assert abs(float(off.mean())) <= ulps * ULP + ULP + 3 * noise, (float(off.mean()) / ULP, noise / ULP)
