"""What the losses' operators refuse before they touch a GPU: the C ABI's checks, and the Python layer's for tensors on the CPU."""

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


def test_token_logprobs(lib):
    def call(logits=P, dtype=0, ld=100, ids=P, ids64=0, lp=P, H=P, st=P, tl=P, ti=P, M=4, V=100, k=5):
        return lib.xkb_token_logprobs(logits, dtype, ld, ids, ids64, lp, H, st, tl, ti, M, V, k, None)

    assert call(M=0) == 0
    for bad in (dict(M=-1), dict(V=0), dict(V=2 ** 31), dict(k=-1), dict(k=65), dict(V=3, k=4), dict(dtype=3), dict(ids64=2), dict(ld=-1),
                dict(M=2 ** 28), dict(logits=None), dict(ids=None), dict(lp=None), dict(H=None), dict(st=None), dict(tl=None), dict(ti=None),
                dict(logits=P + 1), dict(logits=P + 2, dtype=1)):
        assert call(**bad) == -1, bad
        assert b"token_logprobs" in lib.xkb_last_error()


def test_token_logprobs_backward(lib):
    def call(logits=P, dtype=0, ld=104, ids=P, ids64=1, st=P, H=P, glp=P, gh=P, ti=P, gt=P, k=5, out=P, ldg=104, M=4, V=100):
        return lib.xkb_token_logprobs_backward(logits, dtype, ld, ids, ids64, st, H, glp, gh, ti, gt, k, out, ldg, M, V, None)

    assert call(M=0) == 0
    for bad in (dict(M=-1), dict(V=0), dict(k=65), dict(k=-1), dict(dtype=7), dict(ids64=-1), dict(ld=-1), dict(ldg=99), dict(logits=None),
                dict(st=None), dict(out=None), dict(ids=None), dict(H=None), dict(ti=None), dict(out=P + 2), dict(ldg=105),
                dict(logits=P + 1, out=P + 1), dict(M=2 ** 31)):
        assert call(**bad) == -1, bad
        assert b"token_logprobs_backward" in lib.xkb_last_error()


def test_balance_loss(lib):
    def call(g=P, dtype=0, ids=P, mask=None, loss=P, c=P, mean=P, t=P, M=4, E=8, k=2, ws=P, n=1 << 20):
        return lib.xkb_moe_balance_loss(g, dtype, ids, mask, loss, c, mean, t, M, E, k, ws, n, None)

    for bad in (dict(M=-1), dict(E=0), dict(E=1025), dict(k=-1), dict(M=2 ** 30, k=2), dict(dtype=3), dict(g=None), dict(ids=None), dict(loss=None),
                dict(c=None), dict(mean=None), dict(t=None), dict(ws=P + 2)):
        assert call(**bad) == -1, bad
        assert b"moe_balance_loss" in lib.xkb_last_error()
    for bad in (dict(M=2000, ws=None), dict(M=2000, n=16)):
        assert call(**bad) == -3, bad
    size = lib.xkb_moe_balance_loss_workspace_bytes
    assert size(-1, 8) == size(8, 0) == size(8, 1025) == -1
    assert 0 == size(0, 8) == size(512, 8) < size(513, 8) <= size(10 ** 6, 8) == size(10 ** 9, 8)


def test_router_backward(lib):
    def call(g=P, dtype=0, ids=P, gw=P, c=P, t=P, gl=P, mask=None, out=P, M=4, E=8, k=2):
        return lib.xkb_moe_router_backward(g, dtype, ids, gw, 1, c, t, gl, ctypes.c_float(1.0), mask, out, M, E, k, None)

    assert call(M=0) == 0
    for bad in (dict(M=-1), dict(E=0), dict(E=1025), dict(k=-1), dict(dtype=-1), dict(g=None), dict(ids=None), dict(out=None)):
        assert call(**bad) == -1, bad
        assert b"moe_router_backward" in lib.xkb_last_error()


def test_sum_reduce_backward(lib):
    def call(go=P, dtype=0, y=P, w=P, wd=1, gy=P, gw=P, M=4, k=2, H=8):
        return lib.xkb_moe_sum_reduce_backward(go, dtype, y, w, wd, gy, gw, M, k, H, ctypes.c_float(1.0), None)

    assert call(M=0) == 0 and call(k=0) == 0 and call(gy=None, gw=None) == 0
    for bad in (dict(M=-1), dict(k=-1), dict(H=-1), dict(dtype=2), dict(wd=2), dict(w=None), dict(go=None), dict(y=None),
                dict(M=2 ** 30), dict(H=2 ** 28), dict(go=P + 1), dict(y=P + 2, dtype=1, w=P)):
        assert call(**bad) == -1, bad
        assert b"moe_sum_reduce_backward" in lib.xkb_last_error()


def test_misaligned_tensors_and_counts_beyond_64_bits(lib):
    f1 = ctypes.c_float(1.0)

    def logprobs(x=P, dtype=0, ids=P, ids64=0, o=(P, P, P, P, P)):
        return lib.xkb_token_logprobs(x, dtype, 100, ids, ids64, *o, 4, 100, 5, None)

    def logprobs_grad(ids=P, ids64=0, p=(P, P, P, P, P, P), M=4):
        return lib.xkb_token_logprobs_backward(P, 0, 100, ids, ids64, *p[:4], *p[4:], 5, P, 100, M, 100, None)

    def balance(g=P, dtype=0, p=(P, P, P, P, P), M=4, k=2):
        return lib.xkb_moe_balance_loss(g, dtype, p[0], None, *p[1:], M, 8, k, P, 1 << 20, None)

    def router(g=P, dtype=0, p=(P, P, P, P, P), out=P):
        return lib.xkb_moe_router_backward(g, dtype, p[0], p[1], 1, p[2], p[3], p[4], f1, None, out, 4, 8, 2, None)

    def combine(w=P, wd=1, gw=P, M=4, k=2, H=8):
        return lib.xkb_moe_sum_reduce_backward(P, 0, P, w, wd, P, gw, M, k, H, f1, None)

    assert logprobs(ids=P + 4, ids64=1) == -1 and logprobs(ids=P + 2) == -1
    assert logprobs_grad(ids=P + 4, ids64=1) == -1 and logprobs_grad(ids=P + 2) == -1 and logprobs_grad(M=2 ** 62) == -1
    for i in range(6):
        p = tuple(P + 2 if j == i else P for j in range(6))
        assert logprobs_grad(p=p) == -1, i
        if i < 5:
            assert logprobs(o=p[:5]) == balance(p=p[:5]) == router(p=p[:5]) == -1, i
    for dtype, off in ((0, 1), (1, 2), (2, 1)):
        assert balance(g=P + off, dtype=dtype) == router(g=P + off, dtype=dtype) == router(out=P + off, dtype=dtype) == -1
        assert b"misaligned" in lib.xkb_last_error()
    assert balance(M=2 ** 62, k=8) == balance(M=2 ** 40, k=0) == -1
    assert combine(w=P + 2) == combine(gw=P + 2) == combine(w=P + 1, wd=0) == -1
    assert combine(M=2 ** 62, k=8) == combine(M=2 ** 62, k=8, H=0) == -1


def test_there_is_no_cpu_path(lib):
    x, ids, y = torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int32), torch.randn(4, 2, 8)
    for call in (lambda: xkb.token_logprobs(x, ids[:, 0]), lambda: xkb.token_logprobs_backward(x, ids[:, 0], y[0]), lambda: xkb.moe_balance_loss(x, ids),
                 lambda: xkb.moe_router_backward(x, ids, grad_weights=y[:, 0, :2]), lambda: xkb.moe_sum_reduce_backward(x, y),
                 lambda: xka.token_logprobs(x, ids[:, 0]), lambda: xka.moe_balance_loss(x, ids), lambda: xka.topk_softmax(x, 2),
                 lambda: xka.moe_sum_reduce(y)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for call in (lambda: xka.token_logprobs(x.requires_grad_(), ids[:, 0]), lambda: xka.topk_softmax(x, 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    x = x.detach()
    for call in (lambda: xkb.token_logprobs([1.0], ids), lambda: xkb.moe_balance_loss(None, [1]), lambda: xkb.moe_sum_reduce_backward(3, y)):
        with pytest.raises(TypeError):
            call()
