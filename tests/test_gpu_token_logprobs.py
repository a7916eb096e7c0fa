"""token_logprobs against 64 bits: vocabularies around the vector and CTA sizes, rows that lie apart, masked and dead rows, ties,
values that the pass clamps, more candidates than its list holds."""

import math

import pytest
import torch

import xkernels_b200 as xkb
from tests import loss_util as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(x, ids, top_k):
    got = xkb.token_logprobs(x, ids, top_k)
    lp, H, m, l, top, at = ref.token_logprobs(x, ids, top_k)
    assert all(t.dtype == torch.float32 and t.is_contiguous() for t in got[:4]) and got.top_ids.dtype == torch.int32
    assert torch.equal(got.top_ids.long(), at), "top_ids"
    assert torch.equal(got.stats[:, 0].double().nan_to_num(1.0, 2.0, 3.0), m.nan_to_num(1.0, 2.0, 3.0)), "maximum"
    e = ref.sum_error(x.shape[1])
    l0, z = l.nan_to_num(0, 0, 0), (lp - 0).nan_to_num(0, 0, 0).abs()
    ref.assert_near(got.stats[:, 1], l, e + 4 * ref.U24 * l0, "log-sum")
    ref.assert_near(got.logprobs, lp, e + 4 * ref.U24 * (l0 + z), "logprobs")
    ref.assert_near(got.entropy, H, e * (4 + 2 * (l0 + H.nan_to_num(0, 0, 0))), "entropy")
    zt = top.nan_to_num(0, 0, 0).abs()
    ref.assert_near(got.top_logprobs, top, e + 4 * ref.U24 * (l0[:, None] + zt), "top_logprobs")
    return got


def head(M, V, dtype, dev, seed=0, scale=2.0):
    g = torch.Generator(device=dev).manual_seed(1000 * M + V + seed)
    x = (torch.randn(M, V, generator=g, device=dev) * scale).to(dtype)
    ids = torch.randint(0, V, (M,), generator=g, device=dev)
    return x, ids


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 33, 1000, 2047, 2048, 2049, 8191, 32000, 50001, 131072])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes(V, dtype, cuda_device):
    for M, k in ((1, 0), (3, min(V, 20)), (2, min(V, 64)), (1, 1)):
        x, ids = head(M, V, dtype, cuda_device)
        check(x, ids, k)


@pytest.mark.parametrize("M", [1, 2, 73, 74, 75, 147, 149, 300, 600, 1201])
def test_rows(M, cuda_device):
    """Around the numbers of rows where a row gets fewer CTAs."""
    for k in (0, 5):
        x, ids = head(M, 20011, torch.bfloat16, cuda_device)
        check(x, ids, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [297, 593, 1185, 2369, 4000])
def test_many_rows(M, dtype, cuda_device):
    """Around the numbers of rows where a row gets fewer threads, and the widths and alternatives that decide with them."""
    for V, k in ((8, 3), (100, 10), (1000, 0), (2049, 11), (4100, 21), (9001, 22)):
        x, ids = head(M, V, dtype, cuda_device)
        check(x, ids, k)
    x, ids = head(M, 600, dtype, cuda_device)
    x[::3] = -math.inf
    x[1::3, 7:] = torch.finfo(dtype).min
    x[2::6] = 1.0
    x[5::12, 300:] = -math.inf
    x[-1, 5] = math.nan
    for k in (1, 10, 21, 64):
        check(x, ids, k)


@pytest.mark.parametrize("M,k", [(4000, 10), (2000, 20), (1000, 42)])
def test_more_candidates_than_a_small_list_holds(M, k, cuda_device):
    """As below for CTAs of 32, 64 and 128 threads: rows whose large values lie in the vectors of few threads."""
    V = 3000
    g = torch.Generator(device=cuda_device).manual_seed(7)
    n = torch.arange(V, device=cuda_device)
    for step, few in ((32, 9), (64, 19), (128, 40)):
        value = torch.where((n // 4) % step < few, torch.rand(V, generator=g, device=cuda_device) + 9, 0.0)
        x = (value + 0.001 * torch.rand(M, V, generator=g, device=cuda_device))
        check(x, torch.zeros(M, dtype=torch.int64, device=cuda_device), k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,V,pitch", [(0, 1000, 1024), (3, 1001, 1024), (5, 77, 83), (1, 20000, 20003)])
def test_rows_that_lie_apart(dtype, start, V, pitch, cuda_device):
    base, ids = head(9, pitch, dtype, cuda_device)
    x = base[:, start:start + V]
    ids = ids % V
    got = check(x, ids, 5)
    again = xkb.token_logprobs(x.contiguous(), ids.to(torch.int32), 5)
    assert all(torch.equal(a, b) for a, b in zip(got[3:], again[3:])) or torch.allclose(got[3], again[3], atol=1e-5)
    check(base.t().contiguous().t()[:, start:start + V], ids, 3)      # columns apart: copied
    check(base[:1].expand(4, pitch), ids[:4], 3)                      # one row, four times
    check(base[::2], ids[:5] % pitch, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_masked_rows(dtype, V, cuda_device):
    x, ids = head(12, V, dtype, cuda_device)
    low = torch.finfo(dtype).min
    x[0] = -math.inf                                   # nothing left
    x[1, 1:] = -math.inf                               # one token left, the first
    x[2, :-1] = -math.inf                              # one token left, the last
    x[3] = low                                         # all at the type's lowest value: even
    x[4, 3:] = low
    x[5, : V // 2] = -math.inf
    x[6, V // 2:] = low
    x[7] = -math.inf
    x[7, V // 3] = low                                 # the lowest value is all that is left
    x[8] = torch.where(torch.arange(V, device=x.device) % 7 == 0, x[8], -math.inf)
    x[9, ids[9]] = -math.inf                           # the given token is masked
    ids[10], ids[11] = -1, V                           # padding, no token
    check(x, ids, min(V, 20))
    check(x, ids, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 70001])
def test_values_without_a_place(dtype, V, cuda_device):
    x, ids = head(6, V, dtype, cuda_device)
    x[0, V // 2] = math.nan
    x[1, V - 1] = math.inf
    x[2, 0] = -math.nan
    x[3, 3], x[3, 30], x[3, 31] = math.inf, math.nan, math.nan
    x[4] = math.nan
    check(x, ids, 10)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [3e3, -3e3, 5e4, -5e4, 9e5, -9e5, 3e6, -3e6, 1e30, -1e30, 3e38])
def test_large_values(dtype, shift, cuda_device):
    """Far from zero the result is that of the differences, which are exact in 64 bits; the outer ones take the slow pass."""
    if dtype == torch.float16 and abs(shift) > 6e4:
        pytest.skip("not a value of the type")
    g = torch.Generator(device=cuda_device).manual_seed(3)
    step = max(abs(shift), 1.0) * torch.finfo(dtype).eps
    x = (shift - step * torch.randint(0, 9, (5, 3001), generator=g, device=cuda_device).double()).to(dtype)
    x[1, ::2] = -math.inf
    x[2, 1::2] = torch.finfo(dtype).min
    x[3, 5:] = 0.0
    check(x, torch.randint(0, 3001, (5,), generator=g, device=cuda_device), 9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V", [(2, 70001), (700, 3000), (1, 130000)])
def test_ties(dtype, M, V, cuda_device):
    """Equal logits come by ascending id: a whole row, runs of two values, zeros of both signs, a maximum per column block."""
    x, ids = head(M, V, dtype, cuda_device)
    n = torch.arange(V, device=x.device)
    for fill in (torch.zeros(V), (n % 2).float(), (n >= V // 2).float(), (n % 97 == 13).float(), -(n // 4096).float(),
                 torch.where(n % 3 == 0, -0.0, 0.0), ((n * 7919) % 5).float()):
        x[0] = fill.to(x.device, dtype)
        check(x[:2], ids[:2], 64)
        check(x[:2], ids[:2], 3)
    x[:] = 1.5
    check(x, ids, 17)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 600])
def test_more_candidates_than_the_list_holds(dtype, M, cuda_device):
    """All large values fall to the same few threads (vectors 256 apart), distinct, rising or falling."""
    V, N = 131072, 16 // torch.finfo(dtype).bits * 8
    g = torch.Generator(device=cuda_device).manual_seed(5)
    n = torch.arange(V, device=cuda_device)
    mine = (n // N) % 256 < 63
    value = torch.rand(V, generator=g, device=cuda_device) * 64 + 100
    for order in (value, value.sort().values, value.sort(descending=True).values):
        x = torch.where(mine, order, torch.randn(V, generator=g, device=cuda_device)).to(dtype).expand(M, V).contiguous()
        check(x[:2], n[:min(M, 2)].clone(), 64)
        got = xkb.token_logprobs(x, n[:1].expand(M).contiguous(), 64)
        assert bool((got.top_ids == got.top_ids[:1]).all()) and bool((got.top_logprobs == got.top_logprobs[:1]).all())


def test_sharp_and_flat_rows(cuda_device):
    x, ids = head(64, 30000, torch.float32, cuda_device)
    x *= torch.logspace(-6, 2, 64, device=cuda_device)[:, None]
    check(x, ids, 10)
    check(x.sort(dim=1).values, ids, 10)
    check(x.sort(dim=1, descending=True).values, ids, 10)


def test_rows_behind_two_to_the_31(cuda_device):
    M, V = 17000, 131072
    x = torch.zeros(M, V, dtype=torch.bfloat16, device=cuda_device)
    tail, ids = head(3, V, torch.bfloat16, cuda_device)
    x[-3:] = tail
    got = xkb.token_logprobs(x, torch.cat([ids.new_zeros(M - 3), ids]), 4)
    want = xkb.token_logprobs(tail, ids, 4)
    assert torch.equal(got.top_ids[-3:], want.top_ids) and torch.allclose(got.logprobs[-3:], want.logprobs, atol=1e-4)
    assert torch.allclose(got.logprobs[:-3], torch.full((M - 3,), -math.log(V), device=cuda_device), atol=1e-4)


def test_no_rows(cuda_device):
    got = xkb.token_logprobs(torch.zeros(0, 50, device=cuda_device), torch.zeros(0, dtype=torch.int64, device=cuda_device), 5)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 2), (0, 5), (0, 5)]


def test_same_bits(cuda_device):
    x, ids = head(130, 50001, torch.float16, cuda_device)
    a, b = (xkb.token_logprobs(x, ids, 20) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals(cuda_device):
    x, ids = head(4, 100, torch.float32, cuda_device)
    for call, error in ((lambda: xkb.token_logprobs(x.cpu(), ids), RuntimeError), (lambda: xkb.token_logprobs(x, ids.cpu()), RuntimeError),
                        (lambda: xkb.token_logprobs(x.double(), ids), TypeError), (lambda: xkb.token_logprobs(x[0], ids), ValueError),
                        (lambda: xkb.token_logprobs(x, ids[:3]), ValueError), (lambda: xkb.token_logprobs(x, ids.float()), TypeError),
                        (lambda: xkb.token_logprobs(x, None), TypeError), (lambda: xkb.token_logprobs(x[:, :0], ids), ValueError),
                        (lambda: xkb.token_logprobs(x, ids, -1), ValueError), (lambda: xkb.token_logprobs(x, ids, 65), ValueError),
                        (lambda: xkb.token_logprobs(x[:, :5], ids, 6), ValueError)):
        with pytest.raises(error):
            call()
