"""The native call path of the dense operators against their Python form: which calls it serves, the same bits, and that the
others reach the Python form."""

import pytest
import torch

import xkernels_b200 as xkb
from tests.test_gpu_native_loss_calls import _both, served  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,H,V", [(0, 8, 9), (1, 64, 100), (40, 72, 1000), (300, 264, 333)])
def test_linear_cross_entropy(dtype, M, H, V, served, cuda_device):  # noqa: F811
    g = torch.Generator(device=cuda_device).manual_seed(V)
    x, w = torch.randn(M, H, generator=g, device=cuda_device).to(dtype), torch.randn(V, H + 8, generator=g, device=cuda_device).to(dtype)[:, :H]
    gl = torch.randn(M, generator=g, device=cuda_device)
    for labels in (torch.randint(-1, V, (M,), generator=g, device=cuda_device), torch.zeros(M, dtype=torch.int32, device=cuda_device)):
        r = xkb.LinearCrossEntropy(*_both(lambda: xkb.linear_cross_entropy(x, w, labels)))
        _both(lambda: xkb.linear_cross_entropy_backward(x, w, labels, r.stats, gl))
        _both(lambda: xkb.linear_cross_entropy_backward(x, w, labels, r.stats, None, gl, need_grad_weight=False))
        _both(lambda: xkb.linear_cross_entropy_backward(x, w, labels, r.stats, gl, gl, False, True))
    assert served.count("linear_cross_entropy") == 2 and served.count("linear_cross_entropy_backward") == 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,H,I", [(0, 8, 8), (1, 64, 40), (40, 72, 136), (300, 264, 64)])
def test_gated_ffn(dtype, M, H, I, served, cuda_device):  # noqa: F811
    g = torch.Generator(device=cuda_device).manual_seed(M + I)
    x, w13, w2 = (torch.randn(s, generator=g, device=cuda_device).to(dtype) / 8 for s in ((M, H), (2 * I, H), (H, I)))
    for limit in (None, 0.5):
        out, gate_up = _both(lambda: xkb.gated_ffn(x, w13, w2, limit, True))
        _both(lambda: xkb.gated_ffn(x, w13, w2, limit))
        _both(lambda: xkb.gated_ffn_backward(out, x, w13, w2, gate_up, limit))
        _both(lambda: xkb.gated_ffn_backward(out, x, w13, w2, None, limit, True, False, False))
    assert served.count("gated_ffn") == 4 and served.count("gated_ffn_backward") == 4


def test_calls_of_the_python_form(served, cuda_device):  # noqa: F811
    n = lambda *s: torch.randn(*s, device=cuda_device).to(torch.bfloat16)  # noqa: E731
    x, w13, w2, w = n(5, 24), n(16, 24), n(24, 8), n(30, 24)
    labels = torch.zeros(5, dtype=torch.int64, device=cuda_device)
    served.clear()
    want = xkb.gated_ffn(x, w13, w2, 2.0)
    assert served == ["gated_ffn"]
    got = xkb.gated_ffn(x, w13, w2, 2), xkb.gated_ffn(x, w13.t().contiguous().t(), w2, 2.0)       # a whole number, turned weights
    assert served == ["gated_ffn"] and all(torch.equal(a, want) for a in got)
    xkb.linear_cross_entropy(n(5, 23), n(23, 30).t(), labels)                                     # turned weights
    assert served == ["gated_ffn"]
    xkb.linear_cross_entropy(x, w.requires_grad_(), labels)                                       # (a leaf is served: nothing is recorded here)
    assert served == ["gated_ffn", "linear_cross_entropy"]


@pytest.mark.parametrize("H,I", [(23, 9), (24, 9), (23, 16), (257, 130)])
def test_rows_of_no_whole_16_bytes(H, I, served, cuda_device):  # noqa: F811
    g = torch.Generator(device=cuda_device).manual_seed(H + I)
    x, w13, w2, w = (torch.randn(s, generator=g, device=cuda_device).to(torch.bfloat16) / 8 for s in ((37, H), (2 * I, H), (H, I), (60, H)))
    labels = torch.randint(-1, 60, (37,), generator=g, device=cuda_device)
    out, gate_up = _both(lambda: xkb.gated_ffn(x, w13, w2, None, True))
    _both(lambda: xkb.gated_ffn_backward(out, x, w13, w2, gate_up))
    r = xkb.LinearCrossEntropy(*_both(lambda: xkb.linear_cross_entropy(x, w, labels)))
    _both(lambda: xkb.linear_cross_entropy_backward(x, w, labels, r.stats, r.loss))
    assert len(served) == 4
