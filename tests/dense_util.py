"""Plain 64-bit forms of the dense operators (head's cross entropy, gated feed-forward block) and their gradients, each with how far
the kernels' arithmetic may be from it: products in fp32 on the tensor cores, one rounding of the operand of a second product."""

import math

import torch

from tests import loss_util
from tests.loss_util import half_step

U23 = 2.0 ** -23
TINY = {**loss_util.TINY, torch.float64: 0.0}


def acc(K):
    """Relative to the sum of magnitudes: a tensor core cuts off (2^-23) once for each 16 products and sum; a few more are added
    when parts of a sum meet."""
    return (K / 16 + 24) * U23


def rounded(x, err, dtype):
    """How far x, known to err, is off once rounded to dtype."""
    return err + half_step(dtype) * 1.01 * (x.abs() + err) + TINY[dtype]


def product(a, ea, b):
    """(a b^T, its error) of a known to ea and exact b."""
    mag = b.abs().t()
    return a @ b.t(), ea @ mag + acc(a.shape[1]) * ((a.abs() + ea) @ mag)


def clamped(raw, limit):
    gate, up = raw.chunk(2, dim=1)
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(min=-limit, max=limit)
    return gate, up


def gated_ffn(x, w13, w2, limit=None):
    """((out, error), (gate_up, error))"""
    dt = x.dtype
    x, w13, w2 = x.double(), w13.double(), w2.double()
    raw, er = product(x, torch.zeros_like(x), w13)
    gate, up = clamped(raw, limit)
    eg, eu = er.chunk(2, dim=1)
    silu = gate * torch.sigmoid(gate)
    h = silu * up
    # |silu'| < 1.1; the sigmoid and the products of fp32 numbers
    eh = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + 2.0 ** -20 * h.abs()
    return product(h, rounded(h, eh, dt), w2), (raw, er)


def gated_ffn_grad(go, x, w13, w2, raw, limit=None):
    """(value, error) of the gradients of x, w13 and w2, from the saved gate_up"""
    dt = x.dtype
    go, x, w13, w2, raw = (t.double() for t in (go, x, w13, w2, raw))
    gate, up = clamped(raw, limit)
    open_gate, open_up = (raw.chunk(2, dim=1)[0] <= limit, raw.chunk(2, dim=1)[1].abs() <= limit) if limit else (1.0, 1.0)
    s = torch.sigmoid(gate)
    dh, edh = product(go, torch.zeros_like(go), w2.t())
    a, b = up * s * (1 + gate * (1 - s)) * open_gate, gate * s * open_up
    ea, eb = 2.0 ** -19 * up.abs() * s * (1 + gate.abs()), 2.0 ** -20 * (gate * s).abs()
    d13 = torch.cat([dh * a, dh * b], dim=1)
    e13 = torch.cat([edh * (a.abs() + ea) + dh.abs() * ea, edh * (b.abs() + eb) + dh.abs() * eb], dim=1)
    e13 = rounded(d13, e13, dt)
    h = gate * s * up
    eh = rounded(h, 2.0 ** -20 * h.abs(), dt)
    gx = product(d13, e13, w13.t())
    g13 = product(d13.t().contiguous(), e13.t().contiguous(), x.t())
    g2, e2 = product(h.t().contiguous(), eh.t().contiguous(), go.t())
    return gx, g13, (g2.t(), e2.t())


def cross_entropy(x, w, labels):
    """(loss, lse, m, l, error of each)"""
    x, w = x.double(), w.double()
    V = w.shape[0]
    on = labels >= 0
    x = torch.where(on[:, None], x, 0.0)
    z = x @ w.t()
    m = z.max(dim=1).values
    l = torch.logsumexp(z - m[:, None], dim=1)
    given = z.gather(1, labels.long().clamp(0, V - 1)[:, None])[:, 0]
    loss = torch.where(labels >= V, math.nan, m + l - given)
    # logits: parts of 512 K, added up; the sum of exponentials to 2^-19 (terms of 2^-22 and exponents rounded to 2^-24 of them)
    ez = ((512 / 16 + 24 + x.shape[1] / 512) * U23 * (x.abs() @ w.abs().t())).amax(dim=1)
    err = 2 * ez + 2.0 ** -19 + U23 * (m.abs() + l.abs() + given.abs())
    zero = torch.zeros_like(m)
    return tuple(torch.where(on, t, zero) for t in (loss, m + l, m, l)) + (torch.where(on, err, zero),)


def cross_entropy_grad(x, w, labels, stats, g_loss, g_lse, scale=1.0):
    """(value, error) of the gradients of x and w.  scale: what d is multiplied by before it is rounded (fp16)."""
    dt = x.dtype
    V = w.shape[0]
    on = labels >= 0
    x, w, stats = torch.where(on[:, None], x, torch.zeros_like(x)).double(), w.double(), stats.double()
    a = torch.zeros_like(stats[:, 0]) if g_loss is None else torch.where(on, g_loss, 0.0).double()
    b = torch.zeros_like(a) if g_lse is None else torch.where(on, g_lse, 0.0).double()
    z, ez = product(x, torch.zeros_like(x), w)
    e = z - stats[:, :1] - stats[:, 1:]
    p = torch.where(on[:, None], e.exp(), 0.0)
    d = p * (a + b)[:, None]
    at = labels.long().clamp(0, V - 1)
    own = torch.zeros_like(d).scatter_(1, at[:, None], (a * (labels < V))[:, None])
    ed = d.abs() * (ez + 2.0 ** -20 + U23 * (z.abs() + e.abs())) + 2.0 ** -22 * (d.abs() + own.abs())
    d = d - own
    ed = torch.where(on[:, None], rounded(d * scale, ed * scale, dt) / scale, 0.0)
    return product(d, ed, w.t()), product(d.t().contiguous(), ed.t().contiguous(), x.t())


def scale_of(dtype, labels, g_loss, g_lse):
    """The power of two of fp16 gradients: the largest factor comes to 2^10 .. 2^11."""
    if dtype != torch.float16:
        return 1.0
    size = sum(torch.where(labels >= 0, g, 0.0).abs() for g in (g_loss, g_lse) if g is not None)
    top = float(size.max()) if size.numel() else 0.0
    return 2.0 ** (10 - math.floor(math.log2(top))) if 0 < top < math.inf else 1.0
