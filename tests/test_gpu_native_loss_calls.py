"""The native call path of the losses' operators against their Python form: which calls it serves, the same bits, and that the
others reach the Python form."""

import pytest
import torch
from torch.overrides import TorchFunctionMode

import xkernels_b200 as xkb
from xkernels_b200 import _lib

pytestmark = pytest.mark.gpu


class _Passive(TorchFunctionMode):
    """A mode that changes nothing: calls under it belong to the Python form."""

    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _both(fn):
    direct = fn()
    with _Passive():
        python = fn()
    assert type(direct) is type(python)
    direct, python = (r if isinstance(r, tuple) else (r,) for r in (direct, python))
    assert len(direct) == len(python)
    for a, b in zip(direct, python):
        if a is None:
            assert b is None
        else:
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)
    return direct


@pytest.fixture
def served(monkeypatch):
    """Names of the calls that the native path has served."""
    names, calls = [], _lib.load_calls()

    class Watch:
        def __getattr__(self, name):
            def call(*args):
                got = getattr(calls, name)(*args)
                if got is not None:
                    names.append(name)
                return got
            return call

    monkeypatch.setattr(_lib, "_calls", Watch())
    return names


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,V,pitch,k", [(0, 9, 9, 2), (1, 1, 1, 1), (5, 1000, 1008, 20), (7, 2048, 2048, 0)])
def test_token_logprobs(dtype, M, V, pitch, k, served, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = torch.randn(M, pitch, generator=g, device=cuda_device).to(dtype)[:, :V]
    for ids in (torch.randint(-1, V, (M,), generator=g, device=cuda_device), torch.zeros(M, dtype=torch.int32, device=cuda_device)):
        r = xkb.TokenLogprobs(*_both(lambda: xkb.token_logprobs(x, ids, k)))
        gl = torch.randn(M, generator=g, device=cuda_device)
        gt = torch.randn(M, k, generator=g, device=cuda_device)
        _both(lambda: xkb.token_logprobs_backward(x, ids, r.stats, grad_logprobs=gl))
        _both(lambda: xkb.token_logprobs_backward(x, ids, r.stats, r.entropy, gl, gl, r.top_ids, gt))
        _both(lambda: xkb.token_logprobs_backward(x, None, r.stats, r.entropy, grad_entropy=gl))
    assert served.count("token_logprobs") == 2 and served.count("token_logprobs_backward") == 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,E,k", [(0, 8, 2), (1, 1, 1), (300, 60, 6), (2000, 256, 8)])
def test_router(dtype, M, E, k, served, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(M + E)
    x = torch.randn(M, E, generator=g, device=cuda_device).to(dtype)
    ids = torch.rand(M, E, generator=g, device=cuda_device).topk(k, dim=1).indices.to(torch.int32).contiguous()
    gw, mask = torch.randn(M, k, generator=g, device=cuda_device), torch.rand(M, generator=g, device=cuda_device) < 0.5
    for m in (None, mask, mask.to(torch.uint8)):
        b = xkb.BalanceLoss(*_both(lambda: xkb.moe_balance_loss(x, ids, m)))
        for kw in (dict(grad_weights=gw), dict(grad_weights=gw, renormalize=False, counts=b.counts), dict(counts=b.counts, tokens=b.tokens, grad_loss=0.5),
                   dict(counts=b.counts, tokens=b.tokens, grad_loss=b.loss, grad_weights=gw)):
            _both(lambda: xkb.moe_router_backward(x, ids, token_mask=m, **kw))
    assert served.count("moe_balance_loss") == 3 and served.count("moe_router_backward") == 12


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("w_dtype", [None, torch.float32, torch.bfloat16])
def test_combine(dtype, w_dtype, served, cuda_device):
    for M, k, H in ((0, 2, 8), (3, 0, 8), (2, 2, 0), (9, 5, 72), (33, 6, 100)):
        y, go = torch.randn(M, k, H, device=cuda_device).to(dtype), torch.randn(M, H, device=cuda_device).to(dtype)
        w = None if w_dtype is None else torch.rand(M, k, device=cuda_device).to(w_dtype)
        for need in ((True, True), (True, False), (False, True)):
            _both(lambda: xkb.moe_sum_reduce_backward(go, y, w, 0.5, *need))
    assert len(served) == 15


def test_calls_of_the_python_form(served, cuda_device):
    x, ids = torch.randn(6, 40, device=cuda_device), torch.randint(0, 40, (6,), device=cuda_device)
    want = xkb.token_logprobs(x, ids, 3)
    served.clear()
    strided = x.t().contiguous().t()
    for got in (xkb.token_logprobs(strided, ids, 3), xkb.token_logprobs(torch.nn.Parameter(x), ids, 3),
                xkb.token_logprobs(x, torch.stack([ids, ids], 1)[:, 0], 3)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    gl = torch.ones(6, device=cuda_device, dtype=torch.bfloat16)
    xkb.token_logprobs_backward(x, ids, want.stats, grad_logprobs=gl)
    xkb.token_logprobs_backward(x[:, 1:], ids - 1, want.stats, grad_logprobs=gl.float())
    top = torch.zeros(6, 2, dtype=torch.int64, device=cuda_device)
    b = xkb.moe_balance_loss(x, top)
    xkb.moe_router_backward(x, top.int(), counts=b.counts.long())
    xkb.moe_sum_reduce_backward(x, torch.randn(6, 2, 40, device=cuda_device).transpose(0, 1).contiguous().transpose(0, 1))
    xkb.moe_sum_reduce_backward(x, torch.randn(6, 2, 40, device=cuda_device), routed_scaling_factor=2)
    assert served == ["token_logprobs"]      # of the parameter, which is a plain tensor


def test_the_same_refusals(cuda_device):
    x, ids = torch.randn(6, 40, device=cuda_device), torch.randint(0, 40, (6, 2), device=cuda_device, dtype=torch.int32)
    r = xkb.token_logprobs(x, ids[:, 0].contiguous(), 3)
    for call, error in ((lambda: xkb.token_logprobs(x, ids[:, 0].contiguous(), 41), ValueError),
                        (lambda: xkb.token_logprobs(x, ids), ValueError),
                        (lambda: xkb.token_logprobs_backward(x, None, r.stats, grad_logprobs=x[:, 0].contiguous()), ValueError),
                        (lambda: xkb.token_logprobs_backward(x, None, r.stats, grad_entropy=x[:, 0].contiguous()), ValueError),
                        (lambda: xkb.token_logprobs_backward(x, None, r.stats, grad_top_logprobs=x), ValueError),
                        (lambda: xkb.moe_router_backward(x, ids, grad_loss=0.5), ValueError),
                        (lambda: xkb.moe_router_backward(x, ids, grad_weights=x[:, :2].contiguous(), tokens=ids[0, :1].contiguous()), ValueError),
                        (lambda: xkb.moe_balance_loss(torch.zeros(2, 1025, device=cuda_device), ids[:2]), _lib.XkbError)):
        for mode in (None, _Passive()):
            with pytest.raises(error):
                if mode is None:
                    call()
                else:
                    with mode:
                        call()


def test_outputs_are_ordinary_tensors(served, cuda_device):
    """What the native path makes of its own storage: usable, in and out of inference mode, apart from each other."""
    x = torch.randn(8, 100, device=cuda_device)
    ids = torch.randint(0, 100, (8, 2), device=cuda_device, dtype=torch.int32)
    w, y, go = torch.rand(8, 2, device=cuda_device), torch.randn(8, 2, 100, device=cuda_device), torch.randn(8, 100, device=cuda_device)
    def calls():
        r = xkb.token_logprobs(x, ids[:, 0].contiguous(), 3)
        b = xkb.moe_balance_loss(x, ids)
        return [*r, *b, xkb.token_logprobs_backward(x, ids[:, 0].contiguous(), r.stats, grad_logprobs=r.logprobs),
                xkb.moe_router_backward(x, ids, grad_weights=w), *xkb.moe_sum_reduce_backward(go, y, w)]
    want = [t.clone() for t in calls()]
    got = calls()
    for t, v in zip(got, want):
        assert t.device == x.device and t.is_contiguous() and not t.requires_grad and t.grad_fn is None and not t.is_inference()
        assert torch.equal(t, v) and torch.equal(t.cpu(), v.cpu())
    for i, t in enumerate(got):
        t.zero_()
        assert all(torch.equal(u, v) for u, v in zip(got[i + 1:], want[i + 1:]))
        if t.is_floating_point():
            t.requires_grad_()
            (t * 2).sum().backward()
            assert bool((t.grad == 2).all())
    with torch.inference_mode():
        assert all(t.is_inference() and torch.equal(t, v) for t, v in zip(calls(), want))
    a = torch.cuda.memory_allocated(cuda_device)
    calls()
    assert torch.cuda.memory_allocated(cuda_device) == a   # and given back
