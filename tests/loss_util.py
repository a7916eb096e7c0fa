"""Plain 64-bit forms of the losses of a routed model and their gradients, and how far fp32 arithmetic may be from them."""

import math

import torch

U24 = 2.0 ** -24                      # half a step of fp32, relative
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}   # flushed, or half the smallest step


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def log_softmax(x):
    """(ln p, m, l) of rows in 64 bits: m the maximum, l = ln sum exp(x - m); a dead row has ln p = -inf, l = 0; a row with a
    NaN or +inf is NaN."""
    x = x.double()
    m = x.max(dim=1, keepdim=True).values
    dead = m == -math.inf
    z = x - torch.where(dead, 0.0, m)
    l = torch.where(dead, 0.0, z.exp().sum(dim=1, keepdim=True).log())
    return z - l, m, l


def entropy_of(lp):
    p = lp.exp()
    return -torch.where(p > 0, p * lp, torch.where(lp.isnan(), lp, 0.0)).sum(dim=1)


def token_logprobs(x, ids, top_k):
    lp, m, l = log_softmax(x)
    V = x.shape[1]
    given = lp.gather(1, ids.long().clamp(0, V - 1)[:, None])[:, 0]
    given = torch.where(ids < 0, 0.0, torch.where(ids >= V, math.nan, given))
    # (torch sorts a NaN whose sign bit is set below everything)
    order = torch.sort((x.double() + 0.0).masked_fill(x.isnan(), math.nan), dim=1, descending=True, stable=True).indices[:, :top_k]
    return given, entropy_of(lp), m[:, 0], l[:, 0], lp.gather(1, order), order


def sum_error(V):
    """Relative error of a sum of V exponentials: a thread's sum in turn (256 threads), the joins, 2^-22 of an exponential, and the
    rounding of an exponent y, 2^-24 |y| weighted by its 2^y (below 64 in all)."""
    return (V / 256 + 256) * U24


def token_grad(x, ids, entropy_needed, g_lp, g_entropy, top_ids, g_top):
    """(gradient, the magnitude that its errors are relative to)"""
    lp, _, _ = log_softmax(x)
    p = lp.exp()
    M, V = x.shape
    rows = torch.arange(M, device=x.device)
    d, given = torch.zeros_like(p), []
    if g_lp is not None:
        given.append((ids.long(), g_lp))
    if g_top is not None:
        given += list(zip(top_ids.long().unbind(1), g_top.unbind(1)))
    size = torch.zeros(M, 1, dtype=torch.float64, device=x.device)
    own = torch.zeros_like(p)
    for at, g in given:
        g = torch.where(at < 0, 0.0, g.double())
        size += g.abs()[:, None]
        d -= g[:, None] * p
        own[rows, at.clamp(0, V - 1)] += torch.where(at < V, g, 0.0)
    F = size.expand(M, V).clone()
    if g_entropy is not None:
        safe = torch.where(p > 0, lp, 0.0)
        H = -(p * safe).sum(dim=1, keepdim=True)
        d -= g_entropy.double()[:, None] * p * (safe + H)
        F = F + g_entropy.double().abs()[:, None] * (safe.abs() + H)
    # p: exponents |x - m| + |ln p| rounded to fp32, an exponential; the factor: up to 70 terms
    depth = torch.where(p > 0, -lp, 0.0)
    err = p * F * (2.0 ** -21 * (2 + 2 * depth) + 80 * U24) + own.abs() * 80 * U24
    return d + own, err


def softmax_or_zero(x):
    lp, m, _ = log_softmax(x)
    return torch.where(m == -math.inf, 0.0, lp.exp())


def balance(x, ids, mask):
    M, E = x.shape
    k = ids.shape[1]
    on = torch.ones(M, dtype=torch.bool, device=x.device) if mask is None else mask.bool()
    keep = on[:, None] & (ids >= 0) & (ids < E)
    counts = torch.bincount(ids[keep].long(), minlength=E)
    T = int(on.sum())
    p = softmax_or_zero(x)[on]
    mean = p.sum(dim=0) / max(T, 1)
    loss = E * (counts.double() * mean).sum() / (k * T) if T and k else torch.zeros((), dtype=torch.float64, device=x.device)
    return loss, counts, mean, T


def router_grad(x, ids, g_w, renorm, counts=None, tokens=None, g_loss=1.0, mask=None):
    """(gradient, the magnitude that its errors are relative to)"""
    M, E = x.shape
    k = ids.shape[1]
    p = softmax_or_zero(x)
    dp, size = torch.zeros_like(p), torch.zeros_like(p)
    valid = (ids >= 0) & (ids < E)
    at = ids.long().clamp(0, E - 1)
    if g_w is not None:
        sel = p.gather(1, at) * valid
        g = torch.where(valid, g_w.double(), 0.0)
        q, qs = g, g.abs()
        if renorm:
            S = sel.sum(dim=1, keepdim=True)
            q = torch.where(S > 0, (g - (g * sel).sum(dim=1, keepdim=True) / S) / S, 0.0)
            qs = torch.where(S > 0, (g.abs() + (g.abs() * sel).sum(dim=1, keepdim=True) / S) / S, 0.0)
        dp.scatter_add_(1, at, torch.where(valid, q, 0.0))
        size.scatter_add_(1, at, torch.where(valid, qs, 0.0))
    if counts is not None:
        on = torch.ones(M, dtype=torch.bool, device=x.device) if mask is None else mask.bool()
        T = float(M if tokens is None else tokens)
        a = float(g_loss) * E * counts.double() / (k * T * T) if T else torch.zeros(E, dtype=torch.float64, device=x.device)
        dp = dp + a * on[:, None]
        size = size + a.abs() * on[:, None]
    d = p * (dp - (p * dp).sum(dim=1, keepdim=True))
    # probabilities: 2^-21 and the rounding of exponents; sums of up to 1024; divisions
    depth = torch.where(p > 0, -p.clamp(min=1e-300).log(), 0.0)
    err = p * (size + (p * size).sum(dim=1, keepdim=True)) * (2.0 ** -19 + depth * 2.0 ** -23)
    return d, err


def assert_near(got, want, err, what=""):
    """Equal non-finite values, finite ones within ``err`` and half a step of the result's type."""
    assert got.shape == want.shape, f"{what}: {got.shape} vs {want.shape}"
    top = torch.finfo(got.dtype).max          # rounding takes what lies half a step above it to infinity
    want = torch.where(want.abs() >= top * (1 + half_step(got.dtype)), want.sign() * math.inf, want)
    g, fine = got.double(), want.isfinite()
    assert torch.equal(g.isnan(), want.isnan()), f"{what}: NaN in other places"
    other = ~fine & ~want.isnan()
    assert bool((g[other] == want[other]).all()), f"{what}: infinities in other places"
    bound = err + half_step(got.dtype) * want.abs() * 1.01 + TINY[got.dtype]
    off = ((g - want).abs() - bound)[fine]
    if off.numel() and not bool((off <= 0).all()):
        i = int(off.argmax())
        raise AssertionError(f"{what}: {int((~(off <= 0)).sum())} of {off.numel()} outside; worst: got {g[fine][i].item():.9g}, "
                             f"want {want[fine][i].item():.9g}, bound {bound.expand_as(want)[fine][i].item():.3g}")
