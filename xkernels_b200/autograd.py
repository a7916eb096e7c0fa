"""Differentiable forms of the router, the combine, the balance loss, the token log-probabilities, the head's cross entropy and
the gated feed-forward block.

The functions have the arguments and results of their namesakes in :mod:`xkernels_b200.ops`; ``backward()`` runs the
gradient ops there.  First derivatives only.

They are not for stream capture: torch ties the accumulation of a leaf's gradient to the stream that first used the
leaf, and a captured backward pass that meets it on another stream ends the process.  A call that would record a
gradient while its stream is being captured is refused, and so is its backward pass there; a captured step calls the
gradient ops themselves (``ops.moe_router_backward`` and so on), which are ordinary stream-ordered launches.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


def _not_captured(name: str, *inputs) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.is_cuda and t.requires_grad for t in inputs):
        _not_capturing(name)


def _not_capturing(name: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: the differentiable form cannot be captured; call the gradient op of xkernels_b200.ops")


class _TopkSoftmax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gating_output, topk, renormalize):
        w, ids = ops.topk_softmax(gating_output, topk, renormalize)
        ctx.save_for_backward(gating_output, ids)
        ctx.renormalize = renormalize
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return w, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_w, _):
        _not_capturing("topk_softmax")
        if grad_w is None:
            return None, None, None
        gating, ids = ctx.saved_tensors
        return ops.moe_router_backward(gating, ids, grad_weights=grad_w, renormalize=ctx.renormalize), None, None


def topk_softmax(gating_output, topk, renormalize=True):
    """:func:`xkernels_b200.topk_softmax`, differentiable in the logits through the weights."""
    _not_captured("topk_softmax", gating_output)
    return _TopkSoftmax.apply(gating_output, topk, renormalize)


class _SumReduce(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, w, factor):
        out = ops.moe_sum_reduce(y, w, factor)
        # y is needed for w's gradient only, and then only its shape and type remain
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, w)
        ctx.like, ctx.factor = (tuple(y.shape), y.dtype, y.device), factor
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        _not_capturing("moe_sum_reduce")
        if grad_out is None:
            return None, None, None
        y, w = ctx.saved_tensors
        if y is None:
            shape, dtype, device = ctx.like
            y = torch.empty((1,), dtype=dtype, device=device).expand(shape)
        gy, gw = ops.moe_sum_reduce_backward(grad_out, y, w, ctx.factor, need_grad_y=ctx.needs_input_grad[0],
                                             need_grad_w=ctx.needs_input_grad[1])
        return gy, gw, None


def moe_sum_reduce(y, w=None, routed_scaling_factor=1.0):
    """:func:`xkernels_b200.moe_sum_reduce`, differentiable in ``y`` and ``w``."""
    _not_captured("moe_sum_reduce", y, w)
    return _SumReduce.apply(y, w, routed_scaling_factor)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gating_output, topk_ids, token_mask):
        r = ops.moe_balance_loss(gating_output, topk_ids, token_mask)
        ctx.save_for_backward(gating_output, topk_ids, token_mask, r.counts, r.tokens)
        ctx.mark_non_differentiable(r.counts, r.mean_probs, r.tokens)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        _not_capturing("moe_balance_loss")
        if grad_loss is None:
            return None, None, None
        gating, ids, mask, counts, tokens = ctx.saved_tensors
        return ops.moe_router_backward(gating, ids, counts=counts, tokens=tokens, grad_loss=grad_loss, token_mask=mask), None, None


def moe_balance_loss(gating_output, topk_ids, token_mask=None):
    """:func:`xkernels_b200.moe_balance_loss`, its ``loss`` differentiable in the logits (the counts are constants)."""
    _not_captured("moe_balance_loss", gating_output)
    return ops.BalanceLoss(*_BalanceLoss.apply(gating_output, topk_ids, token_mask))


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, token_ids, top_k):
        r = ops.token_logprobs(logits, token_ids, top_k)
        ctx.save_for_backward(logits, token_ids, r.stats, r.entropy, r.top_ids)
        ctx.mark_non_differentiable(r.stats, r.top_ids)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_lp, grad_entropy, _, grad_top, __):
        _not_capturing("token_logprobs")
        if grad_lp is None and grad_entropy is None and grad_top is None:
            return None, None, None
        logits, ids, stats, entropy, top_ids = ctx.saved_tensors
        return ops.token_logprobs_backward(logits, ids, stats, entropy=entropy, grad_logprobs=grad_lp,
                                           grad_entropy=grad_entropy, top_ids=top_ids, grad_top_logprobs=grad_top), None, None


def token_logprobs(logits, token_ids, top_k=0):
    """:func:`xkernels_b200.token_logprobs`, differentiable in the logits through ``logprobs``, ``entropy`` and
    ``top_logprobs``."""
    _not_captured("token_logprobs", logits)
    return ops.TokenLogprobs(*_TokenLogprobs.apply(logits, token_ids, top_k))


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels):
        r = ops.linear_cross_entropy(hidden, weight, labels)
        ctx.save_for_backward(hidden, weight, labels, r.stats)
        ctx.mark_non_differentiable(r.stats)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, grad_lse, _):
        _not_capturing("linear_cross_entropy")
        if grad_loss is None and grad_lse is None:
            return None, None, None
        hidden, weight, labels, stats = ctx.saved_tensors
        gh, gw = ops.linear_cross_entropy_backward(hidden, weight, labels, stats, grad_loss=grad_loss, grad_lse=grad_lse,
                                                   need_grad_hidden=ctx.needs_input_grad[0],
                                                   need_grad_weight=ctx.needs_input_grad[1])
        return gh, gw, None


def linear_cross_entropy(hidden, weight, labels):
    """:func:`xkernels_b200.linear_cross_entropy`, differentiable in ``hidden`` and ``weight`` through ``loss`` and ``lse``."""
    _not_captured("linear_cross_entropy", hidden, weight)
    return ops.LinearCrossEntropy(*_LinearCrossEntropy.apply(hidden, weight, labels))


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, limit, keep):
        got = ops.gated_ffn(x, w13, w2, limit, keep)
        out, gate_up = got if keep else (got, None)
        ctx.save_for_backward(x, w13, w2, gate_up)
        ctx.limit = limit
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        _not_capturing("gated_ffn")
        if grad_out is None:
            return None, None, None, None, None
        x, w13, w2, gate_up = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*ops.gated_ffn_backward(grad_out, x, w13, w2, gate_up, ctx.limit, need[0], need[1], need[2]), None, None)


def gated_ffn(x, w13, w2, swiglu_limit=None, recompute=False):
    """:func:`xkernels_b200.gated_ffn`, differentiable in ``x``, ``w13`` and ``w2``.  ``recompute``: gate and up are not kept for
    the backward pass, which multiplies them once more."""
    _not_captured("gated_ffn", x, w13, w2)
    # (asked here: within forward() gradients are off, and ctx.needs_input_grad is true of a leaf under no_grad as well)
    records = torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, w13, w2))
    return _GatedFfn.apply(x, w13, w2, swiglu_limit, records and not recompute)
