"""B200-native (sm_100a) fused-MoE hot path behind the xkernels operator API.

Public callables (same argument names and meaning as the reference backends):

* :func:`moe_align_block_size`
* :func:`fused_moe_int4_w4a16`
* :func:`fused_moe_mxfp4`
* :func:`moe_sum_reduce`
* :func:`topk_softmax` (the router in front of the path)
* :func:`fused_moe_int4_ffn` (two INT4 GEMMs with SwiGLU between them, one call)

Losses of a routed model and their gradients (no reference counterparts):

* :func:`token_logprobs`, :func:`token_logprobs_backward` (given tokens, entropy, top alternatives)
* :func:`moe_balance_loss` (with per-expert counts), :func:`moe_router_backward` (gating logits)
* :func:`moe_sum_reduce_backward`
* :mod:`xkernels_b200.autograd`: the same as differentiable functions

``plugin.install()`` registers them as the ``backend="cuda"`` cards of an
installed ``xkernels`` package.
"""

from .ops import (  # noqa: F401
    BalanceLoss,
    TokenLogprobs,
    fused_moe_int4_ffn,
    fused_moe_int4_w4a16,
    fused_moe_mxfp4,
    moe_align_block_size,
    moe_balance_loss,
    moe_router_backward,
    moe_sum_reduce,
    moe_sum_reduce_backward,
    token_logprobs,
    token_logprobs_backward,
    topk_softmax,
)

__all__ = [
    "BalanceLoss",
    "TokenLogprobs",
    "fused_moe_int4_ffn",
    "fused_moe_int4_w4a16",
    "fused_moe_mxfp4",
    "moe_align_block_size",
    "moe_balance_loss",
    "moe_router_backward",
    "moe_sum_reduce",
    "moe_sum_reduce_backward",
    "token_logprobs",
    "token_logprobs_backward",
    "topk_softmax",
]
__version__ = "0.1.0"
