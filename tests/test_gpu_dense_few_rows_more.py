"""Gradients of up to 16 rows where the vocabulary goes by in pieces, and captured calls that are replayed over other values."""

import pytest
import torch

import xkernels_b200 as xkb
from tests.test_gpu_dense_few_rows import test_head as check_head
from tests.test_gpu_gated_ffn import BF, HF, no_wait_ran_out  # noqa: F401
from tests.test_gpu_gated_ffn import make as make_block
from tests.test_gpu_linear_cross_entropy import make as make_head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,H,V", [(1, 72, 600_001), (5, 65, 524_289), (16, 40, 1_100_000)])
@pytest.mark.parametrize("dtype,padding", [(BF, 0.0), (HF, 0.4)])
def test_head_in_pieces(M, H, V, dtype, padding, cuda_device):
    """256 rows of 524288 columns are as much of the logits' gradient as is held at a time."""
    check_head(M, H, V, dtype, padding, cuda_device)


@pytest.mark.parametrize("M", [1, 5, 16])
def test_replayed_over_other_values(M, cuda_device):
    x, w13, w2, go = make_block(M, 520, 264, BF, cuda_device)
    h, head, labels = make_head(M, 520, 3001, HF, cuda_device)
    gl = torch.rand(M, device=cuda_device)

    def step():
        out, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
        r = xkb.linear_cross_entropy(h, head, labels)
        return (out, *xkb.gated_ffn_backward(go, x, w13, w2, raw), *xkb.gated_ffn_backward(go, x, w13, w2),
                *xkb.linear_cross_entropy_backward(h, head, labels, r.stats, grad_loss=gl))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        for t in (x, go, h):
            t.copy_(torch.randn(t.shape, generator=g, device=cuda_device))
        gl.uniform_(0.1, 1, generator=g)
        labels.copy_(torch.randint(-seed, 3001, (M,), generator=g, device=cuda_device))
        if seed == 2:
            labels.fill_(-1)       # no row is left
            x[0, 0], go[M - 1, 1] = float("inf"), float("nan")
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, step()):
            assert torch.equal(torch.nan_to_num(a, nan=7.0), torch.nan_to_num(b, nan=7.0)) and torch.equal(a.isnan(), b.isnan())
    assert not got[-1].any() and not got[-2].any()
