"""Performance cases of the dense ends of a routed model: the head's loss from hidden states, and the shared expert.

A case is a dict of plain values; ``listed()`` gives the named ones, ``draw(rng)`` one more of the same ranges.
``prepare`` makes what a program holds before the call, ``run`` is one pass, ``work`` what it cannot do without.

Kinds:
  lce       ``linear_cross_entropy``: the loss of given tokens from hidden states and the head's weight
  lce_grad  ``linear_cross_entropy_backward``: the gradients of both
  ffn       ``gated_ffn``: gate and up projections, SwiGLU, down projection
  ffn_grad  ``gated_ffn_backward``: the gradients of the activations and of both weights

``own`` false: the plain forms, elementary torch operations in fp32.  ``own`` true: the framework's operators.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E = 2                                   # bytes of an element, both types
_MOST_PRODUCTS = 4096 * 7168 * 128000    # M H V of a drawn case: the largest listed one's
_MOST_WEIGHTS = 7168 * 128000            # H V
_MOST_FFN = 8192 * 7168 * 2048           # M H I


def _lce(M, H, V, dtype, padding=0, **name):
    return dict(name, kind="lce", M=M, H=H, V=V, dtype=dtype, padding=padding)


def _lce_grad(M, H, V, dtype, padding=0, lse=False, **name):
    return dict(name, kind="lce_grad", M=M, H=H, V=V, dtype=dtype, padding=padding, lse=lse)


def _ffn(M, H, I, dtype, limit=0.0, save=False, **name):
    return dict(name, kind="ffn", M=M, H=H, I=I, dtype=dtype, limit=limit, save=save)


def _ffn_grad(M, H, I, dtype, limit=0.0, **name):
    return dict(name, kind="ffn_grad", M=M, H=H, I=I, dtype=dtype, limit=limit)


def listed():
    return [
        # scoring one token more: the head's weight streams past one row
        _lce(1, 4096, 50001, "bf16", name="lce_m1"),
        # a short scoring request, odd batch and vocabulary, some prompt tokens without a label
        _lce(77, 2056, 32001, "fp16", padding=13, name="lce_m77_fp16"),
        # a training micro-batch with a large head, padding behind the sequences
        _lce(4096, 7168, 128000, "bf16", padding=409, name="lce_m4096"),
        # its gradient, the largest case
        _lce_grad(4096, 7168, 128000, "bf16", padding=409, name="lce_grad_m4096"),
        # a short batch with a penalty on the log-sum-exp
        _lce_grad(509, 2048, 50001, "fp16", padding=60, lse=True, name="lce_grad_m509_fp16"),
        # one sequence decoding through the shared expert: latency and weight streaming
        _ffn(1, 7168, 2048, "bf16", name="ffn_m1"),
        # a decode batch
        _ffn(64, 7168, 2048, "bf16", name="ffn_m64"),
        # a mixed batch of an odd size through a narrow expert with clamped SwiGLU
        _ffn(509, 4096, 1416, "fp16", limit=10.0, name="ffn_m509_fp16"),
        # a training micro-batch, pre-activations kept for the gradient
        _ffn(8192, 7168, 2048, "bf16", save=True, name="ffn_m8192"),
        # the gradient of a short batch
        _ffn_grad(77, 4096, 1416, "fp16", limit=2.5, name="ffn_grad_m77_fp16"),
        # the gradient of a training micro-batch
        _ffn_grad(4096, 7168, 2048, "bf16", name="ffn_grad_m4096"),
    ]


def _log_int(rng, lo, hi):
    """An integer whose logarithm is spread evenly; an odd one half of the time."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    if rng.random() < 0.5 and v % 2 == 0 and v > lo:
        v -= 1
    return v


def _width(rng, lo, hi):
    """A width: a multiple of 8 as a rule, now and then any."""
    if rng.random() < 0.15:
        return _log_int(rng, lo, hi)
    return 8 * _log_int(rng, -(-lo // 8), hi // 8)


def draw(rng):
    kind = rng.choice(["lce", "lce_grad", "ffn", "ffn_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    H = _width(rng, 64, 7168)
    if kind in ("lce", "lce_grad"):
        V = min(_log_int(rng, 1000, 128000), _MOST_WEIGHTS // H)
        M = _log_int(rng, 1, min(16384, _MOST_PRODUCTS // (H * V)))
        padding = rng.choice([0, M // 10, M // 2])
        if kind == "lce":
            return _lce(M, H, V, dtype, padding=padding)
        return _lce_grad(M, H, V, dtype, padding=padding, lse=rng.random() < 0.3)
    I = _width(rng, 64, 4096)
    M = _log_int(rng, 1, min(16384, _MOST_FFN // (2 * H * I)))
    limit = rng.choice([0.0, 0.0, 2.5, 10.0])
    if kind == "ffn":
        return _ffn(M, H, I, dtype, limit=limit, save=rng.random() < 0.4)
    return _ffn_grad(M, H, I, dtype, limit=limit)


# ---------------------------------------------------------------------------------------------------------------
def _head(case, g, dev):
    """Hidden states in front of a head: most point at the token that follows, more or less; the first ``padding`` rows of a
    shuffled order have no label."""
    M, H, V = case["M"], case["H"], case["V"]
    dt = _DT[case["dtype"]]
    w = torch.randn(V, H, generator=g, device=dev).mul_(1.5 / math.sqrt(H)).to(dt)
    answer = torch.randint(0, V, (M,), generator=g, device=dev)
    x = torch.randn(M, H, generator=g, device=dev)
    x = (x + (1 + 6 * torch.rand(M, 1, generator=g, device=dev)) * w[answer].float()).to(dt)
    other = torch.randint(0, V, (M,), generator=g, device=dev)
    labels = torch.where(torch.rand(M, generator=g, device=dev) < 0.7, answer, other)
    labels[torch.randperm(M, generator=g, device=dev)[: case["padding"]]] = -1
    return x, w, labels


def _expert(case, g, dev):
    M, H, I = case["M"], case["H"], case["I"]
    dt = _DT[case["dtype"]]
    x = torch.randn(M, H, generator=g, device=dev).to(dt)
    w13 = torch.randn(2 * I, H, generator=g, device=dev).mul_(1.2 / math.sqrt(H)).to(dt)
    w2 = torch.randn(H, I, generator=g, device=dev).mul_(1.0 / math.sqrt(I)).to(dt)
    return x, w13, w2


def prepare(case, seed):
    kind, dev = case["kind"], torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 6271 + 29)
    if kind in ("lce", "lce_grad"):
        x, w, labels = _head(case, g, dev)
        state = dict(kind=kind, x=x, w=w, labels=labels)
        if kind == "lce":
            return state
        # what the forward pass left, and gradients of a mean loss under a loss scale
        M = case["M"]
        state["stats"] = torch.where((labels >= 0)[:, None], torch.cat([_stats(p, w) for p in x.split(1024)]), 0.0)
        size = 256.0 / max(M - case["padding"], 1)
        state["g_loss"] = size * (0.5 + torch.rand(M, generator=g, device=dev))
        state["g_lse"] = 0.1 * size * torch.randn(M, generator=g, device=dev) if case["lse"] else None
        return state
    x, w13, w2 = _expert(case, g, dev)
    state = dict(kind=kind, x=x, w13=w13, w2=w2, limit=case["limit"])
    if kind == "ffn":
        state["save"] = case["save"]
        return state
    state["gate_up"] = (x.float() @ w13.float().t()).to(x.dtype)
    state["g_out"] = torch.randn(case["M"], case["H"], generator=g, device=dev).to(x.dtype)
    return state


def _stats(x, w):
    """Row maximum and log of the sum of exponentials, fp32."""
    z = x.float() @ w.float().t()
    m = z.max(dim=1, keepdim=True).values
    return torch.cat([m, (z - m).exp().sum(dim=1, keepdim=True, dtype=torch.float64).log().float()], dim=1)


# ---- the plain forms ------------------------------------------------------------------------------------------
def _plain_lce(s):
    x, labels = s["x"].float(), s["labels"]
    live = labels >= 0
    z = x @ s["w"].float().t()
    m = z.max(dim=1, keepdim=True).values
    l = (z - m).exp().sum(dim=1, keepdim=True).log()
    given = z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    lse = (m + l)[:, 0]
    loss = (m[:, 0] - given) + l[:, 0]
    return torch.where(live, loss, 0.0), torch.where(live, lse, 0.0), torch.where(live[:, None], torch.cat([m, l], dim=1), 0.0)


def _plain_lce_grad(s):
    x, w, labels = s["x"].float(), s["w"].float(), s["labels"]
    live = labels >= 0
    a = torch.where(live, s["g_loss"], 0.0)
    b = a if s["g_lse"] is None else a + torch.where(live, s["g_lse"], 0.0)
    d = x @ w.t()
    d = d.sub_(s["stats"][:, :1]).sub_(s["stats"][:, 1:]).exp_().mul_(b[:, None])
    d.scatter_add_(1, labels.clamp(min=0)[:, None], -a[:, None])
    d = torch.where(live[:, None], d, 0.0)
    return (d @ w).to(s["x"].dtype), (d.t() @ x).to(s["w"].dtype)


def _halves(gate_up, limit):
    g, u = gate_up.chunk(2, dim=1)
    return (g.clamp(max=limit), u.clamp(min=-limit, max=limit)) if limit > 0 else (g, u)


def _plain_ffn(s):
    dt = s["x"].dtype
    gate_up = s["x"].float() @ s["w13"].float().t()
    g, u = _halves(gate_up, s["limit"])
    out = ((g / (1 + (-g).exp()) * u) @ s["w2"].float().t()).to(dt)
    return (out, gate_up.to(dt)) if s["save"] else out


def _plain_ffn_grad(s):
    x, w13, w2, go, limit = s["x"].float(), s["w13"].float(), s["w2"].float(), s["g_out"].float(), s["limit"]
    raw = s["gate_up"].float()
    g, u = _halves(raw, limit)
    dh = go @ w2
    sig = 1 / (1 + (-g).exp())
    dg, du = dh * u * sig * (1 + g * (1 - sig)), dh * g * sig
    if limit > 0:
        g0, u0 = raw.chunk(2, dim=1)
        dg, du = dg * (g0 <= limit), du * (u0.abs() <= limit)
    d13 = torch.cat([dg, du], dim=1)
    dt = s["x"].dtype
    return (d13 @ w13).to(dt), (d13.t() @ x).to(dt), (go.t() @ (g * sig * u)).to(dt)


def run(state):
    s, kind = state, state["kind"]
    if own:
        import xkernels_b200 as xkb

        if kind == "lce":
            return tuple(xkb.linear_cross_entropy(s["x"], s["w"], s["labels"]))
        if kind == "lce_grad":
            return xkb.linear_cross_entropy_backward(s["x"], s["w"], s["labels"], s["stats"], grad_loss=s["g_loss"],
                                                     grad_lse=s["g_lse"])
        if kind == "ffn":
            return xkb.gated_ffn(s["x"], s["w13"], s["w2"], swiglu_limit=s["limit"], save_gate_up=s["save"])
        return xkb.gated_ffn_backward(s["g_out"], s["x"], s["w13"], s["w2"], gate_up=s["gate_up"], swiglu_limit=s["limit"])
    plain = {"lce": _plain_lce, "lce_grad": _plain_lce_grad, "ffn": _plain_ffn, "ffn_grad": _plain_ffn_grad}
    return plain[kind](s)


# ---- in 64 bits -----------------------------------------------------------------------------------------------
def _exact_lce(s):
    loss, lse, stats = [], [], []
    w = s["w"].double()
    for x, t in zip(s["x"].split(512), s["labels"].split(512)):
        z = torch.einsum("mh,vh->mv", x.double(), w)
        top = z.amax(dim=1)
        rest = torch.logsumexp(z - top[:, None], dim=1)
        rows = torch.arange(len(t), device=t.device)
        on = (t >= 0).double()
        lse.append(on * (top + rest))
        loss.append(on * (top + rest - z[rows, t.clamp(min=0)]))
        stats.append(on[:, None] * torch.stack([top, rest], dim=1))
    return torch.cat(loss), torch.cat(lse), torch.cat(stats)


def _exact_lce_grad(s):
    w = s["w"].double()
    gx, gw = [], torch.zeros_like(w)
    parts = [s["x"].split(512), s["labels"].split(512), s["stats"].split(512), s["g_loss"].split(512)]
    extra = torch.zeros_like(s["g_loss"]) if s["g_lse"] is None else s["g_lse"]
    for x, t, st, a, b in zip(*parts, extra.split(512)):
        x, on = x.double(), (t >= 0).double()
        p = torch.exp(torch.einsum("mh,vh->mv", x, w) - st.double().sum(dim=1, keepdim=True))
        d = p * (on * (a.double() + b.double()))[:, None]
        d[torch.arange(len(t), device=t.device), t.clamp(min=0)] -= on * a.double()
        gx.append(torch.einsum("mv,vh->mh", d, w))
        gw += torch.einsum("mv,mh->vh", d, x)
    return torch.cat(gx), gw


def exact(case, seed):
    """``run``'s outputs in 64 bits from the definitions."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "lce":
        return _exact_lce(s)
    if kind == "lce_grad":
        return _exact_lce_grad(s)
    x, w13, w2, top = s["x"].double(), s["w13"].double(), s["w2"].double(), s["limit"] or math.inf
    I = case["I"]
    if kind == "ffn":
        raw = torch.einsum("mh,ih->mi", x, w13)
        gate, up = torch.minimum(raw[:, :I], raw.new_tensor(top)), raw[:, I:].clamp(-top, top)
        out = torch.einsum("mi,hi->mh", gate * torch.sigmoid(gate) * up, w2)
        return (out, raw) if case["save"] else out
    raw, go = s["gate_up"].double(), s["g_out"].double()
    gate, up = torch.minimum(raw[:, :I], raw.new_tensor(top)), raw[:, I:].clamp(-top, top)
    open_, sig = torch.einsum("mh,hi->mi", go, w2), torch.sigmoid(gate)
    slope = sig + gate * sig * torch.sigmoid(-gate)           # of silu
    d = torch.cat([open_ * up * slope * (raw[:, :I] <= top), open_ * gate * sig * (raw[:, I:].abs() <= top)], dim=1)
    return torch.einsum("mi,ih->mh", d, w13), torch.einsum("mi,mh->ih", d, x), torch.einsum("mh,mi->hi", go, gate * sig * up)


def work(case):
    kind, M, H = case["kind"], case["M"], case["H"]
    if kind in ("lce", "lce_grad"):
        V, live = case["V"], M - case["padding"]
        if kind == "lce":
            return {"bytes": _E * H * (live + V) + M * (8 + 16), "flops": 2 * live * H * V}
        # three products: the logits, which nothing kept, and both gradients
        return {"bytes": _E * H * (live + M + 2 * V) + M * (8 + 12 + 4 * case["lse"]), "flops": 6 * live * H * V}
    I = case["I"]
    if kind == "ffn":
        return {"bytes": _E * (2 * M * H + 3 * H * I + 2 * M * I * case["save"]), "flops": 6 * M * H * I}
    return {"bytes": _E * (3 * M * H + 6 * H * I + 2 * M * I), "flops": 12 * M * H * I}
