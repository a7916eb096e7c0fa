"""Gradients of a block whose results leave in different ways within one launch: rows of whole 16 bytes (width H) by copies that run on
behind their warp, others (width I) through the same warp's buffer.  More tiles than pairs of CTAs, so that a warp goes from the one kind
to the other; few rows, so that the next tile's sums are ready when the last copy starts."""

import ctypes

import pytest
import torch

import xkernels_b200 as xkb
from tests import dense_util as du
from tests.loss_util import assert_near
from tests.test_gpu_gated_ffn import BF, HF, make, no_wait_ran_out  # noqa: F401
from xkernels_b200 import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,H,I", [(8, 4096, 1001), (64, 4096, 1001), (64, 2048, 2003), (77, 4096, 1417), (200, 1000, 3001), (300, 4096, 1001),
                                   (512, 4096, 1417), (300, 2049, 2000), (513, 1024, 2500)])
@pytest.mark.parametrize("dtype,limit", [(BF, None), (HF, 0.8)])
def test_rows_of_both_kinds(M, H, I, dtype, limit, cuda_device):
    x, w13, w2, go = make(M, H, I, dtype, cuda_device)
    _, raw = xkb.gated_ffn(x, w13, w2, swiglu_limit=limit, save_gate_up=True)
    want = du.gated_ffn_grad(go, x, w13, w2, raw, limit)
    for need in ((True, True, True), (False, True, True), (True, False, True)):
        first = None
        for _ in range(12):
            got = xkb.gated_ffn_backward(go, x, w13, w2, raw, limit, *need)
            if first is None:
                first = got
                for g, (v, e), what in zip(got, want, ("x", "w13", "w2")):
                    if g is not None:
                        assert_near(g, v, e, "grad " + what)
            assert all(a is b or torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("M", [8, 64, 300])
def test_a_result_that_starts_anywhere(M, cuda_device):
    """Through the C interface: grad_w2 of a width of whole 16 bytes, but starting two bytes behind one."""
    H, I = 2048, 2000
    x, w13, w2, go = make(M, H, I, BF, cuda_device)
    _, raw = xkb.gated_ffn(x, w13, w2, save_gate_up=True)
    want = xkb.gated_ffn_backward(go, x, w13, w2, raw)
    lib = _lib.load()
    need = lib.xkb_gated_ffn_backward_workspace_bytes(M, H, I, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda_device)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for _ in range(12):
        gx, g13 = torch.empty_like(x), torch.empty_like(w13)
        g2 = torch.full((H * I + 2,), 7.0, dtype=BF, device=cuda_device)
        _lib.check(lib.xkb_gated_ffn_backward(p(go), H, _lib.XKB_BF16, p(x), H, p(w13), H, p(w2), I, p(raw), 0.0, p(gx), p(g13),
                                              ctypes.c_void_p(g2.data_ptr() + 2), M, H, I, p(ws), need, ops._stream(cuda_device)),
                   "xkb_gated_ffn_backward")
        assert torch.equal(gx, want[0]) and torch.equal(g13, want[1]) and torch.equal(g2[1:-1].view(H, I), want[2])
        assert g2[0] == 7.0 and g2[-1] == 7.0
