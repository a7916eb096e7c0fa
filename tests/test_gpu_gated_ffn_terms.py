"""The activations of gated_ffn between its products: up to 16 rows in two terms of the type, above that rounded once; and what lies
outside fp16's range."""

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import ops

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def no_wait_ran_out(cuda_device):
    yield
    ops.check_status(cuda_device)


def differ(M, I, dtype, dev):
    """Rows whose result is the difference of two activations, 40 (1 + e) - 40, the first of which has more bits than a term: silu(40)
    is 40 in fp32, and every number here but that one is exact.  The columns that differ lie at the ends of the block."""
    e = torch.finfo(dtype).eps
    w13, w2 = torch.zeros(2 * I, 8, device=dev), torch.zeros(8, I, device=dev)
    w13[[0, I - 1], 0] = 40
    w13[[I, 2 * I - 1], 1] = 1
    w13[I, 2] = e
    w2[:, 0], w2[:, I - 1] = 1, -1
    x = torch.zeros(M, 8, device=dev)
    x[:, :3] = 1
    return x.to(dtype), w13.to(dtype), w2.to(dtype), 40 * e


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("I", [2, 72, 1001, 2048])
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 300])
def test_two_terms_up_to_16_rows(M, I, dtype, cuda_device):
    x, w13, w2, want = differ(M, I, dtype, cuda_device)
    out = xkb.gated_ffn(x, w13, w2).double()
    once = (torch.tensor(40 * (1 + torch.finfo(dtype).eps), dtype=torch.float64).to(dtype).double() - 40).item()
    assert once != want
    assert bool((out == (want if M <= 16 else once)).all())


@pytest.mark.parametrize("M", [4, 300])
def test_activations_beyond_the_range_of_fp16(M, cuda_device):
    """They become infinite, as a cast does, and so does what they are added up to."""
    x = torch.zeros(M, 8, device=cuda_device, dtype=HF)
    x[:, 0] = 1
    x[1, 1] = 1
    w13, w2 = torch.zeros(4, 8, device=cuda_device, dtype=HF), torch.full((8, 2), 2.0 ** -10, device=cuda_device, dtype=HF)
    w13[[0, 2], 0], w13[[0, 2], 1] = 200, 100          # 200 * 200 = 40000 in most rows, 300 * 300 = 90000 in row 1
    out = xkb.gated_ffn(x, w13, w2)
    assert out[1].isinf().all() and bool((out[[i for i in range(M) if i != 1]] == 40000 / 1024).all())
