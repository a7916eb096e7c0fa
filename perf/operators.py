"""Performance cases of the losses of a routed model and their gradients.

A case is a dict of plain values; ``listed()`` gives the named ones, ``draw(rng)`` one more of the same ranges.
``prepare`` makes what a program holds before the call, ``run`` is one pass, ``work`` what it cannot do without.

Kinds:
  logprobs       ``token_logprobs``: log-probabilities of given tokens, entropy, top alternatives
  logprobs_grad  ``token_logprobs_backward``: the gradient of the head's logits
  balance        ``moe_balance_loss``: balance loss and per-expert counts of a routing
  router_grad    ``moe_router_backward``: the gradient of the gating logits, from the routing weights and the balance loss
  combine_grad   ``moe_sum_reduce_backward``: the gradients of the expert rows and of the routing weights

``own`` false: the plain forms, elementary torch operations in fp32.  ``own`` true: the framework's operators.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
_ESIZE = {"bf16": 2, "fp32": 4, "fp16": 2}
_MOST_BYTES = 1 << 30          # of logits in a drawn case
_MOST_SORTED = 1 << 26         # logits of a drawn case with top alternatives


def _logprobs(M, V, dtype, top, masked=False, **name):
    return dict(name, kind="logprobs", M=M, V=V, dtype=dtype, top=top, masked=masked)


def _logprobs_grad(M, V, dtype, entropy, top=0, **name):
    return dict(name, kind="logprobs_grad", M=M, V=V, dtype=dtype, entropy=entropy, top=top)


def _balance(M, E, k, dtype, masked=False, **name):
    return dict(name, kind="balance", M=M, E=E, k=k, dtype=dtype, masked=masked)


def _router_grad(M, E, k, dtype, renorm=True, balance=True, masked=False, **name):
    return dict(name, kind="router_grad", M=M, E=E, k=k, dtype=dtype, renorm=renorm, balance=balance, masked=masked)


def _combine_grad(M, k, H, dtype, w_dtype="fp32", factor=1.0, **name):
    return dict(name, kind="combine_grad", M=M, k=k, H=H, dtype=dtype, w_dtype=w_dtype, factor=factor)


def listed():
    return [
        # one sequence decoding, the answer's log-probability and 20 alternatives per step: latency counts
        _logprobs(1, 128000, "bf16", 20, name="logprobs_m1"),
        # a decode batch whose sampler works on fp32 logits; some rows under a grammar that allows few tokens or none
        _logprobs(64, 128000, "fp32", 5, masked=True, name="logprobs_m64_fp32"),
        # prompt log-probabilities of a scoring request, odd batch and vocabulary
        _logprobs(509, 50001, "fp16", 20, name="logprobs_m509"),
        # a training micro-batch: token loss and entropy, the largest head
        _logprobs(4096, 128000, "bf16", 0, name="logprobs_m4096"),
        # its gradient, with an entropy bonus
        _logprobs_grad(4096, 128000, "bf16", True, name="logprobs_grad_m4096"),
        # distillation on a few alternatives of a short fp32 batch
        _logprobs_grad(77, 32001, "fp32", False, top=8, name="logprobs_grad_m77_fp32"),
        # the router of a training micro-batch
        _balance(16384, 256, 8, "bf16", name="balance_m16384"),
        # a short padded batch, fp32 gating
        _balance(333, 48, 4, "fp32", masked=True, name="balance_m333_fp32"),
        # both gradients of the gating logits, training micro-batch
        _router_grad(16384, 256, 8, "bf16", name="router_grad_m16384"),
        # raw weights, no balance loss, odd sizes
        _router_grad(77, 60, 6, "fp32", renorm=False, balance=False, name="router_grad_m77_fp32"),
        # the combine of a training micro-batch, the largest case
        _combine_grad(8192, 8, 7168, "bf16", name="combine_grad_m8192"),
        # a short batch of fp32 rows, scaled routing
        _combine_grad(37, 6, 2056, "fp32", factor=2.5, name="combine_grad_m37_fp32"),
    ]


def _log_int(rng, lo, hi):
    """An integer whose logarithm is spread evenly; an odd one half of the time."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    if rng.random() < 0.5 and v % 2 == 0 and v > lo:
        v -= 1
    return v


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs_grad", "balance", "router_grad", "combine_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    es = _ESIZE[dtype]
    if kind == "logprobs":
        V = _log_int(rng, 1000, 128000)
        top = rng.choice([0, 0, 1, 5, 20, 64])
        most = min(_MOST_BYTES // (V * es), 16384)
        if top:
            most = max(1, min(most, _MOST_SORTED // V))
        return _logprobs(_log_int(rng, 1, most), V, dtype, top, masked=rng.random() < 0.25)
    if kind == "logprobs_grad":
        V = _log_int(rng, 1000, 128000)
        top = rng.choice([0, 0, 5, 16])
        most = min(_MOST_BYTES // (V * es), 16384)
        if top:
            most = max(1, min(most, _MOST_SORTED // V))
        return _logprobs_grad(_log_int(rng, 1, most), V, dtype, rng.random() < 0.5, top=top)
    if kind == "balance":
        E = _log_int(rng, 4, 512)
        return _balance(_log_int(rng, 1, 65536), E, rng.randint(1, min(E, 10)), dtype, masked=rng.random() < 0.5)
    if kind == "router_grad":
        E = _log_int(rng, 4, 512)
        return _router_grad(_log_int(rng, 1, 65536), E, rng.randint(1, min(E, 10)), dtype, renorm=rng.random() < 0.6,
                            balance=rng.random() < 0.7, masked=rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    H, k = _log_int(rng, 64, 8192), rng.randint(1, 10)
    most = max(1, (_MOST_BYTES // 2) // (H * k * _ESIZE[dtype]))
    return _combine_grad(_log_int(rng, 1, min(most, 32768)), k, H, dtype, w_dtype=rng.choice(["fp32", "fp32", "bf16"]),
                         factor=rng.choice([1.0, 2.5]))


# ---------------------------------------------------------------------------------------------------------------
def _head(case, g, dev):
    """Logits of a language-model head: a tilt over the vocabulary shared by all rows, noise, and in most rows a token that
    stands out more or less; the given tokens are mostly those."""
    M, V = case["M"], case["V"]
    x = torch.randn(M, V, generator=g, device=dev).mul_(2.0).add_(torch.randn(V, generator=g, device=dev).mul_(1.5))
    answer = torch.randint(0, V, (M,), generator=g, device=dev)
    x.scatter_add_(1, answer[:, None], 4 + 12 * torch.rand(M, 1, generator=g, device=dev))
    other = torch.randint(0, V, (M,), generator=g, device=dev)
    ids = torch.where(torch.rand(M, generator=g, device=dev) < 0.7, answer, other)
    return x, ids


def _gating(case, g, dev):
    """Gating logits of a router with a mild preference for some experts, and the routing that follows from them."""
    M, E, k = case["M"], case["E"], case["k"]
    x = torch.randn(M, E, generator=g, device=dev) + 0.5 * torch.randn(E, generator=g, device=dev)
    x = x.to(_DT[case["dtype"]])
    p = torch.softmax(x.double(), dim=-1)
    ids = torch.sort(p, dim=-1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
    mask = None
    if case["masked"]:
        mask = torch.rand(M, generator=g, device=dev) < 0.8
        mask[0] = True
    return x, ids, mask


def prepare(case, seed):
    kind, dev = case["kind"], torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)
    if kind in ("logprobs", "logprobs_grad"):
        M, V = case["M"], case["V"]
        x, ids = _head(case, g, dev)
        if case.get("masked"):     # a grammar: all tokens, about one in fifty, three, or none are allowed, by row
            how = torch.randint(0, 8, (M, 1), generator=g, device=dev)
            some = torch.rand(M, V, generator=g, device=dev) < 0.02
            few = torch.zeros(M, V, dtype=torch.bool, device=dev)
            few.scatter_(1, torch.randint(0, V, (M, 3), generator=g, device=dev), True)
            x.masked_fill_(~((how < 4) | ((how < 6) & some) | ((how == 6) & few)), -math.inf)
        x = x.to(_DT[case["dtype"]])
        state = dict(kind=kind, x=x, ids=ids, top=case["top"])
        if kind == "logprobs":
            return state
        ids[torch.rand(M, generator=g, device=dev) < 0.1] = -1           # padding behind sequences
        # what the forward pass left: row maximum and log-sum, entropy, the alternatives' ids
        parts = [_forward64(p, t, case["top"]) for p, t in zip(x.split(256), ids.split(256))]
        stats, entropy, top_ids = (torch.cat([p[i] for p in parts]) for i in (2, 1, 4))
        state.update(stats=stats.float(), entropy=entropy.float() if case["entropy"] else None,
                     top_ids=top_ids if case["top"] else None)
        state["g_lp"] = torch.randn(M, generator=g, device=dev) / M
        state["g_entropy"] = 0.05 * torch.randn(M, generator=g, device=dev) / M if case["entropy"] else None
        state["g_top"] = torch.randn(M, case["top"], generator=g, device=dev) / M if case["top"] else None
        return state
    if kind == "balance":
        x, ids, mask = _gating(case, g, dev)
        return dict(kind=kind, x=x, ids=ids, mask=mask)
    if kind == "router_grad":
        x, ids, mask = _gating(case, g, dev)
        state = dict(kind=kind, x=x, ids=ids, mask=mask, renorm=case["renorm"], counts=None, tokens=None, g_loss=None)
        state["g_w"] = torch.randn(case["M"], case["k"], generator=g, device=dev)
        if case["balance"]:
            state["counts"], state["tokens"] = _counts(ids, mask, case["E"])
            state["g_loss"] = 0.01 + torch.rand((), generator=g, device=dev)
        return state
    M, k, H, dt = case["M"], case["k"], case["H"], _DT[case["dtype"]]
    y = torch.randn(M, k, H, generator=g, device=dev).to(dt)
    w = torch.softmax(torch.randn(M, k, generator=g, device=dev), dim=-1).to(_DT[case["w_dtype"]])
    go = (torch.randn(M, H, generator=g, device=dev) / math.sqrt(H)).to(dt)
    return dict(kind=kind, go=go, y=y, w=w, factor=case["factor"])


# ---- the plain forms ------------------------------------------------------------------------------------------
def _counts(ids, mask, E):
    """How many slots of counted tokens each expert has, and how many tokens count."""
    on = torch.ones(ids.shape[0], dtype=torch.bool, device=ids.device) if mask is None else mask
    flat = ids.long().clamp(0, E - 1)
    keep = (on[:, None] & (ids >= 0) & (ids < E)).to(torch.int32)
    counts = torch.zeros(E, dtype=torch.int32, device=ids.device).scatter_add_(0, flat.reshape(-1), keep.reshape(-1))
    return counts, on.sum().to(torch.int32)


def _plain_logprobs(s):
    x, ids, top = s["x"].float(), s["ids"], s["top"]
    m = x.max(dim=-1, keepdim=True).values
    z = x - torch.where(m == -math.inf, 0.0, m)
    e = z.exp()
    S = e.sum(dim=-1, keepdim=True)
    live = S > 0
    l = torch.where(live, S, 1.0).log()
    T = (e * torch.where(e > 0, z, 0.0)).sum(dim=-1, keepdim=True)
    entropy = torch.where(live, l - T / torch.where(live, S, 1.0), 0.0)
    lp = (z - l).gather(1, ids.clamp(min=0)[:, None])[:, 0]
    out = [torch.where(ids >= 0, lp, 0.0), entropy[:, 0], torch.cat([m, l], dim=1)]
    if top:
        v, at = torch.sort(x, dim=-1, descending=True, stable=True)
        at = at[:, :top]
        out += [(z - l).gather(1, at), at.to(torch.int32)]
    return out


def _plain_logprobs_grad(s):
    x, ids, m, l = s["x"].float(), s["ids"], s["stats"][:, :1], s["stats"][:, 1:]
    logp = x - m - l
    p = torch.where(m == -math.inf, 0.0, logp.exp())
    on = ids >= 0
    g = torch.where(on, s["g_lp"], 0.0)
    G = g[:, None] if s["g_top"] is None else (g + s["g_top"].sum(dim=1))[:, None]
    if s["g_entropy"] is not None:
        G = G + s["g_entropy"][:, None] * (torch.where(p > 0, logp, 0.0) + s["entropy"][:, None])
    d = -p * G
    d.scatter_add_(1, ids.clamp(min=0)[:, None], g[:, None])
    if s["g_top"] is not None:
        d.scatter_add_(1, s["top_ids"].long(), s["g_top"])
    return d.to(s["x"].dtype)


def _plain_balance(s):
    x, ids, mask = s["x"].float(), s["ids"], s["mask"]
    E, k = x.shape[1], ids.shape[1]
    counts, tokens = _counts(ids, mask, E)
    z = x - x.max(dim=-1, keepdim=True).values
    p = z.exp()
    p = p / p.sum(dim=-1, keepdim=True)
    if mask is not None:
        p = p * mask[:, None]
    T = tokens.clamp(min=1).double()
    mean = p.sum(dim=0, dtype=torch.float64) / T        # a sum over all tokens
    loss = E * (counts.double() / (k * T) * mean).sum()
    return loss.float(), counts, mean.float(), tokens


def _plain_router_grad(s):
    x, ids, mask = s["x"].float(), s["ids"].long(), s["mask"]
    E, k = x.shape[1], ids.shape[1]
    z = x - x.max(dim=-1, keepdim=True).values
    p = z.exp()
    p = p / p.sum(dim=-1, keepdim=True)
    q = s["g_w"]
    if s["renorm"]:
        sel = p.gather(1, ids)
        S = sel.sum(dim=1, keepdim=True)
        q = (q - (q * sel).sum(dim=1, keepdim=True) / S) / S
    dp = torch.zeros_like(p).scatter_add_(1, ids, q)
    if s["counts"] is not None:
        T = s["tokens"].float()
        a = s["g_loss"] * E * s["counts"].float() / (k * T * T)
        dp = dp + (a if mask is None else a * mask[:, None])
    return (p * (dp - (p * dp).sum(dim=1, keepdim=True))).to(s["x"].dtype)


def _plain_combine_grad(s):
    go, y, w, f = s["go"].float(), s["y"], s["w"], s["factor"]
    gy = (f * w.float())[:, :, None] * go[:, None, :]
    gw = f * (go[:, None, :] * y.float()).sum(dim=-1)
    return gy.to(y.dtype), gw.to(w.dtype)


def run(state):
    s, kind = state, state["kind"]
    if own:
        import xkernels_b200 as xkb

        if kind == "logprobs":
            r = xkb.token_logprobs(s["x"], s["ids"], s["top"])
            return [r.logprobs, r.entropy, r.stats] + ([r.top_logprobs, r.top_ids] if s["top"] else [])
        if kind == "logprobs_grad":
            return xkb.token_logprobs_backward(s["x"], s["ids"], s["stats"], entropy=s["entropy"], grad_logprobs=s["g_lp"],
                                               grad_entropy=s["g_entropy"], top_ids=s["top_ids"],
                                               grad_top_logprobs=s["g_top"])
        if kind == "balance":
            r = xkb.moe_balance_loss(s["x"], s["ids"], token_mask=s["mask"])
            return r.loss, r.counts, r.mean_probs, r.tokens
        if kind == "router_grad":
            return xkb.moe_router_backward(s["x"], s["ids"], grad_weights=s["g_w"], renormalize=s["renorm"],
                                           counts=s["counts"], tokens=s["tokens"], grad_loss=s["g_loss"],
                                           token_mask=s["mask"])
        return xkb.moe_sum_reduce_backward(s["go"], s["y"], s["w"], s["factor"])
    plain = {"logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad, "balance": _plain_balance,
             "router_grad": _plain_router_grad, "combine_grad": _plain_combine_grad}
    return plain[kind](s)


# ---- in 64 bits -----------------------------------------------------------------------------------------------
def _log_softmax64(x):
    """(log-probabilities, maximum, log-sum) of each row; a row of nothing but -inf has -inf, -inf and 0"""
    m = x.amax(dim=1, keepdim=True)
    l = torch.logsumexp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m), dim=1, keepdim=True)
    l = torch.where(torch.isinf(m), torch.zeros_like(l), l)
    return torch.where(torch.isinf(m), torch.full_like(x, -math.inf), x - m - l), m, l


def _forward64(x, ids, top):
    lp, m, l = _log_softmax64(x.double())
    given = torch.where(ids < 0, 0.0, lp.gather(1, ids.clamp(min=0).unsqueeze(1)).squeeze(1))
    entropy = -torch.special.xlogy(lp.exp(), lp.exp()).sum(dim=1)
    at = torch.argsort(-x.double(), dim=1, stable=True)[:, :top] if top else ids.new_zeros(ids.shape[0], 0)
    return given, entropy, torch.cat([m, l], dim=1), lp.gather(1, at), at.to(torch.int32)


def _head_grad64(s, i, j):
    x, ids = s["x"][i:j].double(), s["ids"][i:j]
    lp, _, _ = _log_softmax64(x)
    p = lp.exp()
    d = torch.zeros_like(p)
    rows = torch.arange(j - i, device=x.device)
    given = [(ids, s["g_lp"][i:j])]
    if s["g_top"] is not None:
        given += list(zip(s["top_ids"][i:j].long().unbind(1), s["g_top"][i:j].unbind(1)))
    for at, g in given:
        g = g.double() * (at >= 0)
        d -= g[:, None] * p
        d[rows, at.clamp(min=0)] += g
    if s["g_entropy"] is not None:       # dH/dx = -p (ln p - sum p ln p)
        plogp = torch.special.xlogy(p, p)
        d -= s["g_entropy"][i:j].double()[:, None] * (plogp - p * plogp.sum(dim=1, keepdim=True))
    return d


def exact(case, seed):
    """``run``'s outputs in 64 bits from the definitions; whole numbers have no such value."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "logprobs":
        parts = [_forward64(x, t, case["top"]) for x, t in zip(s["x"].split(256), s["ids"].split(256))]
        out = [torch.cat([p[i] for p in parts]) for i in range(4)]
        return out + [None] if case["top"] else out[:3]
    if kind == "logprobs_grad":
        M = case["M"]
        return torch.cat([_head_grad64(s, i, min(i + 256, M)) for i in range(0, M, 256)])
    if kind == "combine_grad":
        gy, gw = [], []
        for go, y, w in zip(s["go"].split(512), s["y"].split(512), s["w"].split(512)):
            gy.append(torch.einsum("mk,mh->mkh", w.double() * s["factor"], go.double()))
            gw.append(torch.einsum("mh,mkh->mk", go.double(), y.double()) * s["factor"])
        return torch.cat(gy), torch.cat(gw)
    p = torch.softmax(s["x"].double(), dim=1)
    M, E = p.shape
    k = s["ids"].shape[1]
    on = torch.ones(M, dtype=torch.float64, device=p.device) if s["mask"] is None else s["mask"].double()
    chosen = torch.nn.functional.one_hot(s["ids"].long(), E).double()            # [M, k, E]
    share = torch.einsum("mke,m->e", chosen, on) / (k * on.sum())
    if kind == "balance":
        mean = torch.einsum("me,m->e", p, on) / on.sum()
        return E * (share @ mean), None, mean, None
    gw = s["g_w"].double()
    if case["renorm"]:
        sel = torch.einsum("mke,me->mk", chosen, p)
        total = sel.sum(dim=1, keepdim=True)
        gw = gw / total - (gw * sel).sum(dim=1, keepdim=True) / total**2
    dp = torch.einsum("mke,mk->me", chosen, gw)
    if case["balance"]:
        dp = dp + s["g_loss"].double() * E * torch.outer(on, share) / on.sum()
    jac = p * dp
    return jac - p * jac.sum(dim=1, keepdim=True)


def work(case):
    kind, M, e = case["kind"], case["M"], _ESIZE[case["dtype"]]
    if kind == "logprobs":
        return {"bytes": M * (case["V"] * e + 8 + 16 + 8 * case["top"]), "flops": 6 * M * case["V"]}
    if kind == "logprobs_grad":
        return {"bytes": M * (2 * case["V"] * e + 8 + 8 + 4 + 8 * case["entropy"] + 8 * case["top"]),
                "flops": 6 * M * case["V"]}
    if kind == "balance":
        return {"bytes": M * (case["E"] * e + 4 * case["k"] + case["masked"]) + 8 * case["E"] + 8, "flops": 6 * M * case["E"]}
    if kind == "router_grad":
        return {"bytes": M * (2 * case["E"] * e + 8 * case["k"] + case["masked"]) + 4 * case["E"] * case["balance"],
                "flops": 8 * M * case["E"]}
    k, H = case["k"], case["H"]
    return {"bytes": M * ((2 * k + 1) * H * e + 2 * k * _ESIZE[case["w_dtype"]]), "flops": 3 * M * k * H}
