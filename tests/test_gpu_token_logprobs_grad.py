"""token_logprobs_backward against the formula in 64 bits and against differences of the 64-bit forward form."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from tests import loss_util as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def case(M, V, dtype, dev, top=0, entropy=True, seed=0):
    g = torch.Generator(device=dev).manual_seed(M + 31 * V + seed)
    x = (torch.randn(M, V, generator=g, device=dev) * 2).to(dtype)
    ids = torch.randint(0, V, (M,), generator=g, device=dev)
    kw = dict(g_lp=torch.randn(M, generator=g, device=dev), g_entropy=torch.randn(M, generator=g, device=dev) if entropy else None,
              g_top=torch.randn(M, top, generator=g, device=dev) if top else None)
    return x, ids, kw


def check(x, ids, top, g_lp=None, g_entropy=None, g_top=None):
    _, H, m, l, _, at = ref.token_logprobs(x, ids, top)
    stats = torch.stack([m, l], dim=1).float()
    at = at.to(torch.int32)
    got = xkb.token_logprobs_backward(x, ids, stats, entropy=H.float(), grad_logprobs=g_lp, grad_entropy=g_entropy,
                                      top_ids=at, grad_top_logprobs=g_top)
    assert got.dtype == x.dtype and got.shape == x.shape and (got.stride(1) == 1 or x.shape[1] == 1)
    want, err = ref.token_grad(x, ids, True, g_lp, g_entropy, at, g_top)
    if g_lp is not None:
        want[ids >= x.shape[1]] = math.nan
    ref.assert_near(got, want, err, "gradient")
    return got


@pytest.mark.parametrize("V", [1, 7, 8, 9, 1000, 2049, 8193, 50001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes(V, dtype, cuda_device):
    for M, top, entropy in ((1, 0, False), (5, min(V, 8), True), (3, min(V, 64), False), (700, 0, True)):
        x, ids, kw = case(M, V, dtype, cuda_device, top, entropy)
        check(x, ids, top, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_each_gradient_alone(dtype, cuda_device):
    x, ids, kw = case(6, 3001, dtype, cuda_device, 4)
    for name in kw:
        check(x, ids, 4, **{name: kw[name]})
    check(x, ids.to(torch.int32), 4, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,V,pitch", [(0, 1000, 1024), (3, 1001, 1024), (5, 77, 83), (0, 1001, 1003)])
def test_rows_that_lie_apart(dtype, start, V, pitch, cuda_device):
    base, ids, kw = case(9, pitch, dtype, cuda_device, 5)
    x, ids = base[:, start:start + V], ids % V
    check(x, ids, 5, **kw)
    check(base.t().contiguous().t()[:, start:start + V], ids, 5, **kw)
    check(base[:1].expand(9, pitch), ids, 5, **kw)
    check(base[3:4, start:], ids[:1], 5, **{k: v[:1] for k, v in kw.items()})


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_padded_and_shared(dtype, cuda_device):
    V = 5003
    x, ids, kw = case(10, V, dtype, cuda_device, 20)
    x[0] = -math.inf
    x[1, 5:] = -math.inf                     # fewer live tokens than alternatives
    x[2, V // 2:] = torch.finfo(dtype).min
    x[3] = torch.finfo(dtype).min
    ids[4] = -1
    kw["g_lp"][4] = math.nan                 # of padding: not looked at
    ids[5] = int(x[5].float().argmax())      # the given token is an alternative too
    ids[6] = V
    x[7, ids[7]] = -math.inf
    ids[2] %= V // 2
    check(x, ids, 20, **kw)
    check(x, ids, 20, g_lp=kw["g_lp"])


def test_the_same_column_again(cuda_device):
    """Alternatives may name a column twice, and none."""
    x, ids, _ = case(3, 500, torch.float32, cuda_device)
    at = torch.tensor([[4, 4, 4, 9], [-1, 3, 3, -1], [0, 499, 500, 0]], dtype=torch.int32, device=cuda_device)
    g = torch.randn(3, 4, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1))
    ids[0] = 4
    g_lp = torch.ones(3, device=cuda_device)
    _, _, m, l, _, _ = ref.token_logprobs(x, ids, 0)
    got = xkb.token_logprobs_backward(x, ids, torch.stack([m, l], dim=1).float(), grad_logprobs=g_lp, top_ids=at, grad_top_logprobs=g)
    want, err = ref.token_grad(x, ids, False, g_lp, None, at, g)
    want[2] = math.nan                       # 500 is no column
    ref.assert_near(got, want, err)
    wide = at.long()
    wide[1, 0], wide[1, 3] = -(2 ** 33), 2 ** 32 + 3      # nor are these, one no token and one behind the row
    got = xkb.token_logprobs_backward(x, ids, torch.stack([m, l], dim=1).float(), grad_logprobs=g_lp, top_ids=wide, grad_top_logprobs=g)
    want[1] = math.nan
    ref.assert_near(got, want, err)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [-5e4, 9e5, -3e6, 1e30])
def test_large_values(dtype, shift, cuda_device):
    if dtype == torch.float16 and abs(shift) > 6e4:
        pytest.skip("not a value of the type")
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = (shift - abs(shift) * torch.finfo(dtype).eps * torch.randint(0, 9, (4, 301), generator=g, device=cuda_device).double()).to(dtype)
    x[1, ::2] = -math.inf
    _, ids, kw = case(4, 301, dtype, cuda_device, 3)
    check(x, ids, 3, **kw)


def test_rows_with_nan(cuda_device):
    x, ids, kw = case(4, 999, torch.bfloat16, cuda_device)
    x[1, 7], x[2, 9] = math.nan, math.inf
    r = xkb.token_logprobs(x, ids)
    got = xkb.token_logprobs_backward(x, ids, r.stats, entropy=r.entropy, grad_logprobs=kw["g_lp"], grad_entropy=kw["g_entropy"])
    assert bool(got[1:3].isnan().all()) and bool(got[[0, 3]].isfinite().all())


def test_against_differences(cuda_device):
    """sum of dx v against (f(x + h v) - f(x - h v)) / 2h of the 64-bit forms, whose error is about h^2 + 2^-52 / h."""
    x, ids, kw = case(5, 700, torch.float32, cuda_device, 6)
    r = xkb.token_logprobs(x, ids, 6)
    got = xkb.token_logprobs_backward(x, ids, r.stats, entropy=r.entropy, grad_logprobs=kw["g_lp"], grad_entropy=kw["g_entropy"],
                                      top_ids=r.top_ids, grad_top_logprobs=kw["g_top"]).double()

    def f(z):
        lp, _, _ = ref.log_softmax(z)
        out = kw["g_lp"].double() * lp.gather(1, ids[:, None])[:, 0] + kw["g_entropy"].double() * ref.entropy_of(lp)
        return out + (kw["g_top"].double() * lp.gather(1, r.top_ids.long())).sum(dim=1)

    _, err = ref.token_grad(x, ids, True, kw["g_lp"], kw["g_entropy"], r.top_ids, kw["g_top"])
    g = torch.Generator(device=cuda_device).manual_seed(2)
    for _ in range(4):
        v = torch.randn(5, 700, generator=g, device=cuda_device, dtype=torch.float64)
        h = 1e-5
        want = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
        bound = ((err + ref.U24 * got.abs()) * v.abs()).sum(dim=1) + 1e-8 * v.abs().sum(dim=1)
        assert bool((((got * v).sum(dim=1) - want).abs() <= bound).all())


def test_rows_behind_two_to_the_31(cuda_device):
    M, V = 17000, 131072
    x = torch.zeros(M, V, dtype=torch.bfloat16, device=cuda_device)
    tail, ids, kw = case(3, V, torch.bfloat16, cuda_device)
    x[-3:] = tail
    ids = torch.cat([ids.new_full((M - 3,), -1), ids])
    g = torch.cat([torch.zeros(M - 3, device=cuda_device), kw["g_lp"]])
    r = xkb.token_logprobs(x, ids)
    got = xkb.token_logprobs_backward(x, ids, r.stats, grad_logprobs=g)
    want = xkb.token_logprobs_backward(tail, ids[-3:], r.stats[-3:], grad_logprobs=kw["g_lp"])
    assert torch.equal(got[-3:], want) and not bool(got[:-3].any())


def test_no_rows_and_refusals(cuda_device):
    x, ids, kw = case(4, 100, torch.float32, cuda_device, 3)
    r = xkb.token_logprobs(x, ids, 3)
    assert xkb.token_logprobs_backward(x[:0], ids[:0], r.stats[:0], grad_logprobs=kw["g_lp"][:0]).shape == (0, 100)
    f = xkb.token_logprobs_backward
    for call, error in ((lambda: f(x, ids, r.stats), ValueError), (lambda: f(x, None, r.stats, grad_logprobs=kw["g_lp"]), ValueError),
                        (lambda: f(x, ids, r.stats, grad_entropy=kw["g_entropy"]), ValueError),
                        (lambda: f(x, ids, r.stats, grad_top_logprobs=kw["g_top"]), ValueError),
                        (lambda: f(x, ids, r.stats[:3], grad_logprobs=kw["g_lp"]), ValueError),
                        (lambda: f(x, ids, r.stats, grad_logprobs=kw["g_lp"][:3]), ValueError),
                        (lambda: f(x.double(), ids, r.stats, grad_logprobs=kw["g_lp"]), TypeError),
                        (lambda: f(x, ids, r.stats.cpu(), grad_logprobs=kw["g_lp"]), RuntimeError),
                        (lambda: f(x, ids, r.stats, top_ids=r.top_ids[:, :2], grad_top_logprobs=kw["g_top"]), ValueError),
                        (lambda: f(x, ids, r.stats, top_ids=r.top_ids.float(), grad_top_logprobs=kw["g_top"]), TypeError),
                        (lambda: f(x, ids, r.stats, top_ids=ids[:, None].expand(4, 65), grad_top_logprobs=x[:, :65]), ValueError)):
        with pytest.raises(error):
            call()
