"""token_logprobs_backward of rows without a live logit (all -inf): no probability, but a token that is no column makes the row NaN, as
it does the forward call's log-probability, and as it does in any other row."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import autograd as xka

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("V", [1, 9, 5003, 50001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_token_behind_the_row(V, dtype, cuda_device):
    """Rows: dead and ordinary ones, each with a token of the row, padding, and tokens behind it."""
    x = torch.randn(8, V, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(V)).to(dtype)
    x[:4] = -math.inf
    ids = torch.tensor([V - 1, -1, V, 2 ** 40] * 2, device=cuda_device)
    g_lp = torch.full((8,), 0.5, device=cuda_device)
    r = xkb.token_logprobs(x, ids, 1)
    assert r.logprobs.isnan().tolist() == [False, False, True, True] * 2
    for kw in (dict(), dict(entropy=r.entropy, grad_entropy=g_lp), dict(top_ids=r.top_ids, grad_top_logprobs=torch.zeros(8, 1, device=cuda_device))):
        got = xkb.token_logprobs_backward(x, ids, r.stats, grad_logprobs=g_lp, **kw)
        assert bool(got[[2, 3, 6, 7]].isnan().all())
        assert bool(got[[0, 1, 4, 5]].isfinite().all())
        want = torch.zeros(V, dtype=dtype, device=cuda_device)     # p = 0: what the column was given
        want[V - 1] = 0.5
        assert torch.equal(got[0], want) and not bool(got[1].any())
    # alternatives that are no columns
    at = torch.tensor([[V], [-1], [0], [V]] * 2, dtype=torch.int32, device=cuda_device)
    got = xkb.token_logprobs_backward(x, ids, r.stats, top_ids=at, grad_top_logprobs=g_lp[:, None])
    assert got.isnan().all(dim=1).tolist() == got.isnan().any(dim=1).tolist() == [True, False, False, True] * 2


def test_through_autograd(cuda_device):
    x = torch.full((2, 300), -math.inf, device=cuda_device, requires_grad=True)
    r = xka.token_logprobs(x, torch.tensor([299, 300], device=cuda_device))
    assert r.logprobs.isnan().tolist() == [False, True]
    r.logprobs.sum().backward()
    assert bool(x.grad[0].isfinite().all()) and bool(x.grad[1].isnan().all())
