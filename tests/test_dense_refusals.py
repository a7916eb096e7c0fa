"""What the dense operators refuse before they touch a GPU: the C ABI's checks, and the Python layer's for tensors on the CPU."""

import ctypes

import pytest
import torch

import xkernels_b200 as xkb
from xkernels_b200 import _lib
from xkernels_b200 import autograd as xka


@pytest.fixture(scope="module")
def lib():
    from xkernels_b200.build import build

    build()
    return _lib.load()


P = 4096   # an address that is never used: every call here is refused before its launch
BIG = 1 << 50


def test_gated_ffn(lib):
    def call(x=P, ldx=64, dtype=0, w13=P, ld13=64, w2=P, ld2=40, out=P, gu=P, M=4, H=64, I=40, ws=P, n=BIG):
        return lib.xkb_gated_ffn(x, ldx, dtype, w13, ld13, w2, ld2, ctypes.c_float(0.0), out, gu, M, H, I, ws, n, None)

    assert call(M=0) == 0 and call(M=0, x=None, out=None) == 0
    for bad in (dict(dtype=1), dict(dtype=3), dict(M=-1), dict(H=0), dict(I=0), dict(M=2 ** 28), dict(H=2 ** 24), dict(I=2 ** 24), dict(x=None), dict(w13=None),
                dict(w2=None), dict(x=P + 8), dict(w13=P + 2), dict(w2=P + 8), dict(ldx=65), dict(ld13=60), dict(ld13=56), dict(ld2=32), dict(ldx=2 ** 32),
                dict(out=None), dict(out=P + 1), dict(gu=P + 1)):
        assert call(**bad) == -1, bad
        assert b"gated_ffn" in lib.xkb_last_error()
    for bad in (dict(ws=None), dict(n=16), dict(ws=P + 16)):
        assert call(**bad) == -3, bad
    size = lib.xkb_gated_ffn_workspace_bytes
    assert size(-1, 8, 8) == size(1, 0, 8) == size(1, 8, 0) == -1 and size(0, 8, 8) == 0 < size(1, 8, 8) < size(1000, 8, 8)


def test_gated_ffn_backward(lib):
    def call(go=P, ldg=64, dtype=2, x=P, ldx=64, w13=P, ld13=64, w2=P, ld2=40, gu=P, gx=P, g13=P, g2=P, M=4, H=64, I=40, ws=P, n=BIG):
        return lib.xkb_gated_ffn_backward(go, ldg, dtype, x, ldx, w13, ld13, w2, ld2, gu, ctypes.c_float(1.0), gx, g13, g2, M, H, I, ws, n, None)

    assert call(gx=None, g13=None, g2=None) == 0 and call(M=0, g13=None, g2=None) == 0
    for bad in (dict(dtype=1), dict(M=-1), dict(H=0), dict(I=0), dict(go=None), dict(x=None), dict(w13=None), dict(w2=None), dict(go=P + 8), dict(ldg=60),
                dict(ldx=72 + 1), dict(ld2=36), dict(gx=P + 1), dict(g13=P + 1), dict(g2=P + 1), dict(gu=P + 1)):
        assert call(**bad) == -1, bad
        assert b"gated_ffn_backward" in lib.xkb_last_error()
    for bad in (dict(ws=None), dict(n=16), dict(ws=P + 16)):
        assert call(**bad) == -3, bad
    size = lib.xkb_gated_ffn_backward_workspace_bytes
    assert size(-1, 8, 8, 0) == -1 and 0 < size(9, 8, 8, 0) < size(9, 8, 8, 1)


def test_linear_cross_entropy(lib):
    def call(x=P, ldx=64, dtype=0, w=P, ldw=64, ids=P, ids64=1, loss=P, lse=P, st=P, M=4, H=64, V=100, ws=P, n=BIG):
        return lib.xkb_linear_cross_entropy(x, ldx, dtype, w, ldw, ids, ids64, loss, lse, st, M, H, V, ws, n, None)

    assert call(M=0) == 0
    for bad in (dict(dtype=1), dict(M=-1), dict(H=0), dict(V=0), dict(M=2 ** 28), dict(V=2 ** 28), dict(H=2 ** 24), dict(x=None), dict(w=None), dict(ids=None),
                dict(x=P + 1), dict(w=P + 8), dict(ldw=60), dict(ldw=56), dict(ldx=-1), dict(ids64=2), dict(ids=P + 4), dict(ids64=0, ids=P + 2), dict(loss=None),
                dict(lse=None), dict(st=None), dict(loss=P + 2), dict(lse=P + 2), dict(st=P + 2)):
        assert call(**bad) == -1, bad
        assert b"linear_cross_entropy" in lib.xkb_last_error()
    for bad in (dict(ws=None), dict(n=16), dict(ws=P + 16)):
        assert call(**bad) == -3, bad
    size = lib.xkb_linear_cross_entropy_workspace_bytes
    assert size(-1, 8, 8) == size(1, 0, 8) == size(1, 8, 0) == -1 and size(0, 8, 8) == 0 < size(1, 8, 8) < size(5000, 8, 8)


def test_linear_cross_entropy_backward(lib):
    def call(x=P, ldx=64, dtype=0, w=P, ldw=64, ids=P, ids64=1, st=P, gl=P, gs=P, gx=P, gw=P, M=4, H=64, V=100, ws=P, n=BIG):
        return lib.xkb_linear_cross_entropy_backward(x, ldx, dtype, w, ldw, ids, ids64, st, gl, gs, gx, gw, M, H, V, ws, n, None)

    assert call(gx=None, gw=None) == 0 and call(M=0, gw=None) == 0
    for bad in (dict(dtype=1), dict(M=-1), dict(H=0), dict(V=0), dict(x=None), dict(w=None), dict(ids=None), dict(st=None), dict(gl=None, gs=None), dict(st=P + 2),
                dict(gl=P + 2), dict(gs=P + 2), dict(gx=P + 1), dict(gw=P + 1), dict(w=P + 8), dict(ldw=60), dict(ids=P + 4)):
        assert call(**bad) == -1, bad
        assert b"linear_cross_entropy_backward" in lib.xkb_last_error()
    for bad in (dict(ws=None), dict(n=16), dict(ws=P + 16)):
        assert call(**bad) == -3, bad
    size = lib.xkb_linear_cross_entropy_backward_workspace_bytes
    # one piece of the logits' gradient, whatever the vocabulary
    assert size(4096, 64, 128000) < (256 << 20) + 16 * 4096 * 64 + 4096 * 64 * 4 * 32 + (64 << 20)
    assert size(-1, 8, 8) == -1 and size(0, 8, 8) == 0


def test_lay_out_rows(lib):
    arrays = lambda t, *v: (t * 4)(*v)  # noqa: E731
    ok = dict(f=arrays(ctypes.c_void_p, P, P), ld=arrays(ctypes.c_int64, 9, 9), rows=arrays(ctypes.c_int64, 0, 0), cols=arrays(ctypes.c_int64, 9, 3),
              to=arrays(ctypes.c_void_p, P, P), count=2)

    def call(**kw):
        a = {**ok, **kw}
        return lib.xkb_lay_out_rows(a["f"], a["ld"], a["rows"], a["cols"], a["to"], a["count"], None)

    assert call() == 0 and call(count=0, f=None) == 0
    for bad in (dict(count=5), dict(count=-1), dict(f=None), dict(to=None), dict(rows=arrays(ctypes.c_int64, 0, -1)), dict(cols=arrays(ctypes.c_int64, 0, 3)),
                dict(ld=arrays(ctypes.c_int64, -1, 9)), dict(rows=arrays(ctypes.c_int64, 0, 1), f=arrays(ctypes.c_void_p, P, None)),
                dict(rows=arrays(ctypes.c_int64, 1, 0), to=arrays(ctypes.c_void_p, P + 1, P))):
        assert call(**bad) == -1, bad
        assert b"lay_out_rows" in lib.xkb_last_error()


def test_there_is_no_cpu_path(lib):
    x, w, labels = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(9, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    w13, w2, st, g = torch.zeros(12, 8, dtype=torch.bfloat16), torch.zeros(8, 6, dtype=torch.bfloat16), torch.zeros(4, 2), torch.zeros(4)
    for call in (lambda: xkb.linear_cross_entropy(x, w, labels), lambda: xkb.linear_cross_entropy_backward(x, w, labels, st, g),
                 lambda: xkb.gated_ffn(x, w13, w2), lambda: xkb.gated_ffn_backward(x, x, w13, w2), lambda: xka.linear_cross_entropy(x, w, labels),
                 lambda: xka.gated_ffn(x, w13, w2), lambda: xka.gated_ffn(x.clone().requires_grad_(), w13, w2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for call in (lambda: xkb.linear_cross_entropy([1.0], w, labels), lambda: xkb.gated_ffn(3, w13, w2)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
def test_arguments(lib, cuda_device):
    n = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=cuda_device)  # noqa: E731
    x, w, labels, w13, w2 = n(4, 8), n(9, 8), n(4, t=torch.int64), n(12, 8), n(8, 6)
    st, g = n(4, 2, t=torch.float32), n(4, t=torch.float32)
    f32, f16 = torch.float32, torch.float16
    for call in (lambda: xkb.linear_cross_entropy(x, n(9, 7), labels), lambda: xkb.linear_cross_entropy(x[0], w, labels),
                 lambda: xkb.linear_cross_entropy(x, w, labels[:3]), lambda: xkb.linear_cross_entropy(x, n(0, 8), labels),
                 lambda: xkb.linear_cross_entropy_backward(x, w, labels, st), lambda: xkb.linear_cross_entropy_backward(x, w, labels, st[:3], g),
                 lambda: xkb.linear_cross_entropy_backward(x, w, labels, st, g[:2]), lambda: xkb.gated_ffn(x, n(11, 8), w2),
                 lambda: xkb.gated_ffn(x, w13, n(7, 6)), lambda: xkb.gated_ffn(x, w13, n(8, 5)), lambda: xkb.gated_ffn(x[0], w13, w2),
                 lambda: xkb.gated_ffn_backward(n(3, 8), x, w13, w2), lambda: xkb.gated_ffn_backward(x, x, w13, w2, n(4, 11))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: xkb.linear_cross_entropy(x.to(f32), w.to(f32), labels), lambda: xkb.linear_cross_entropy(x, w.to(f16), labels),
                 lambda: xkb.linear_cross_entropy(x, w, g), lambda: xkb.gated_ffn(x.to(f32), w13.to(f32), w2.to(f32)),
                 lambda: xkb.gated_ffn(x, w13.to(f16), w2), lambda: xkb.gated_ffn(x, w13, w2.to(f16)),
                 lambda: xkb.gated_ffn_backward(x.to(f16), x, w13, w2), lambda: xkb.gated_ffn_backward(x, x, w13, w2, n(4, 12, t=f16)),
                 lambda: xkb.linear_cross_entropy(x, None, labels), lambda: xkb.linear_cross_entropy(x, w, None), lambda: xkb.gated_ffn(x, None, w2)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: xkb.linear_cross_entropy(x, w.cpu(), labels), lambda: xkb.gated_ffn(x, w13, w2.cpu())):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
