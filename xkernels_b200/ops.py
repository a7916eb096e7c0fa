"""Host side of the ops: argument checks, output allocation, one C-ABI call.

The callables keep the parameter names of the reference backends because the
reference's ``verify`` harness calls a card as ``fn(**inputs)``
(src/xkernels/verify.py:213-222 with names from
src/xkernels/registry/input_gen.py:68-72,84-103,138-159).  PyTorch is used for
device memory and the current stream only; all arithmetic happens in
``libxkb200.so``.
"""

from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.XKB_BF16, torch.float32: _lib.XKB_F32}
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def _require_cuda(name: str, *tensors) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: expected torch.Tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(
                f"{name}: the sm_100a backend needs CUDA tensors (got device {t.device}); "
                "there is no CPU path"
            )
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"{name}: tensors live on different devices ({dev} vs {t.device})")
    return dev


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# The small ops take less time on the device than a call spends in Python, so a call asks for the raw
# stream (0.1 us; a Stream object 1 us) and enters a device only if another one is current (2 us).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_CURRENT = contextlib.nullcontext()


def _stream(dev: torch.device) -> int:
    if _raw_stream is not None and dev.index is not None:
        return _raw_stream(dev.index)
    return torch.cuda.current_stream(dev).cuda_stream


def _on(dev: torch.device):
    return _CURRENT if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


@functools.lru_cache(maxsize=512)
def _bytes(query: str, *dims) -> int:
    """A workspace size query of the library (arithmetic on the dimensions only)."""
    return int(getattr(_lib.load(), query)(*dims))


_retired: list[torch.Tensor] = []


def get_workspace(dev: torch.device, nbytes: int, tag: int = 0) -> torch.Tensor:
    """Grow-only per-device scratch buffer shared by calls on one stream.

    Calls that overlap on different streams of one device must pass distinct
    ``tag`` values (or serialise): the buffer holds the routing and the fp32
    partial rows of the call in flight.  When a larger call needs a new buffer the old one is kept
    alive (until :func:`release_workspaces`): a CUDA graph captured earlier, or work still queued
    on another stream, may hold its address.  A caller that wants to own the memory passes
    ``workspace=`` to the fused ops instead.
    """
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), tag)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _retired.append(buf)
        size = max(int(nbytes), 1 << 20)
        if buf is not None:
            size = max(size, 2 * buf.numel())        # geometric growth bounds what the retired buffers hold
        buf = torch.empty(size, dtype=torch.uint8, device=dev)
        _workspaces[key] = buf
    return buf


def _caller_workspace(workspace, fits: bool, nbytes_at_capacity: int, dev: torch.device, nbytes: int) -> torch.Tensor:
    """The scratch memory of one fused call.

    ``workspace`` None: this package's per-device buffer.  A CUDA ``uint8`` tensor: used as it is
    (ValueError if it is too small or misaligned).  One of the reference's workspace objects
    (``MoeInt4Workspace`` / ``MoeMxfp4Workspace``, src/xkernels/ops/moe/workspace.py:159-289):
    when its ``matches()`` accepted the call (``fits``), the call's scratch lives in a buffer that is
    created once, sized for the object's capacity, and kept ON the object, so every call through
    that object sees the same addresses - which is what the reference's workspaces are for (CUDA
    graph capture, workspace.py:32-35).  The layout of the kernels here (routing, fp32 slot rows,
    gathered activations) is not the reference's, so its ``scratch`` / ``combine_out`` / ``act``
    tensors are not reinterpreted.  When ``matches()`` refused, the object is ignored and the call
    falls back to the per-device buffer, as the reference falls back to fresh allocations
    (triton/moe_int4_kernel.py:550-558)."""
    if workspace is None:
        return get_workspace(dev, nbytes)
    if isinstance(workspace, torch.Tensor):
        if workspace.dtype != torch.uint8 or not workspace.is_cuda or workspace.device != dev or not workspace.is_contiguous():
            raise ValueError("workspace tensor must be a contiguous uint8 tensor on the inputs' device")
        if workspace.numel() < nbytes or workspace.data_ptr() % 256:
            raise ValueError(f"workspace tensor needs {nbytes} bytes at a 256-byte aligned address "
                             f"(got {workspace.numel()} bytes)")
        return workspace
    if not fits:
        return get_workspace(dev, nbytes)
    buf = getattr(workspace, "_xkb200_scratch", None)
    if buf is None or buf.numel() < nbytes or buf.device != dev:
        buf = torch.empty(max(int(nbytes_at_capacity), int(nbytes)), dtype=torch.uint8, device=dev)
        workspace._xkb200_scratch = buf
    return buf


def check_workspace_status(workspace) -> None:
    """As :func:`check_status`, for a call that was given ``workspace=``."""
    buf = workspace if isinstance(workspace, torch.Tensor) else getattr(workspace, "_xkb200_scratch", None)
    if buf is None:
        return
    with torch.cuda.device(buf.device):
        _lib.check(_lib.load().xkb_workspace_status(buf.data_ptr(), _stream(buf.device)), "xkb_workspace_status")


def check_status(dev=None, tag: int = 0) -> None:
    """Synchronise and raise if a kernel of the last fused call on ``dev``, or of any dense one there (:func:`gated_ffn`,
    :func:`linear_cross_entropy` and their gradients), gave up a bounded wait (the tcgen05 kernels never spin without a
    limit; they record a status word instead)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if dev is None else torch.device(dev)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), tag)
    buf = _workspaces.get(key)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().xkb_dense_status(_stream(dev)), "xkb_dense_status")
        if buf is not None:
            _lib.check(_lib.load().xkb_workspace_status(buf.data_ptr(), _stream(dev)), "xkb_workspace_status")


def release_workspaces() -> None:
    """Drop the per-device buffers (only when no captured graph or queued work still uses them)."""
    _workspaces.clear()
    _retired.clear()


# ---------------------------------------------------------------------------
def moe_align_block_size(topk_ids, block_size, num_experts, truncate=True, workspace=None,
                         expert_map=None):
    """Sort/pad routed token-slots into per-expert blocks on the GPU.

    Same contract as ``moe_align_block_size_ref``
    (src/xkernels/ops/moe/w4a16.py:53-101): returns ``(sorted_token_ids
    [M*top_k + (E+1)*(block-1)], expert_ids, num_tokens_post_padded [1])``, all
    int32, bit-exact with the reference including the unused tails.
    ``truncate=True`` trims ``expert_ids`` to the used blocks and therefore
    reads ``num_tokens_post_padded`` back (one host sync); ``truncate=False`` is
    sync-free.  ``expert_map`` gives the expert-parallel form of
    ``moe_align_block_size_ep`` (w4a16.py:104-155): ``num_experts`` is then the
    local expert count and non-local slots are dropped.
    """
    if workspace is None and expert_map is None:
        got = (_lib._calls or _lib.load_calls()).moe_align_block_size(topk_ids, block_size, num_experts)
        if got is not None:
            if type(got) is int:
                _lib.check(got, "xkb_moe_align_block_size")
            if not truncate:
                return got
            sorted_ids, expert_ids, num_post = got
            return sorted_ids, expert_ids[: max(int(num_post.item()) // block_size, 1)], num_post
    lib = _lib.load()
    dev = _require_cuda("moe_align_block_size", topk_ids, expert_map)
    block_size, num_experts = int(block_size), int(num_experts)
    if block_size <= 0:
        raise ValueError("block_size must be > 0")
    ids = topk_ids.reshape(-1)
    if ids.dtype != torch.int32:
        ids = ids.to(torch.int32)
    ids = ids.contiguous()
    numel = ids.numel()
    emap = None
    if expert_map is not None:
        emap = expert_map.to(device=dev, dtype=torch.int32).contiguous()
    max_pad = numel + (num_experts + 1) * (block_size - 1)
    max_blocks = -(-max_pad // block_size)
    # A reference MoeAlignWorkspace (src/xkernels/ops/moe/workspace.py:85-151) that matches the call:
    # the three outputs are written INTO its buffers (address-stable, the reference's contract at
    # triton/align_kernel.py:198-213,245-250) and this kernel's own scratch is kept on the object.
    use_ws = False
    if workspace is not None and hasattr(workspace, "matches") and topk_ids.dim() == 2:
        use_ws = bool(workspace.matches(topk_ids.shape[0], topk_ids.shape[1], num_experts, block_size, device=dev))
    with _on(dev):
        ws_bytes = _bytes("xkb_moe_align_workspace_bytes", numel, num_experts)
        if use_ws:
            sorted_ids, expert_ids, num_post = workspace.sorted_ids, workspace.expert_ids, workspace.num_post
            if max_blocks == 0:
                expert_ids[:1].zero_()
            ws = getattr(workspace, "_xkb200_scratch", None)
            if ws is None or ws.numel() < ws_bytes:
                cap = _bytes("xkb_moe_align_workspace_bytes", max(workspace.sorted_ids.numel(), numel), num_experts)
                ws = torch.empty(max(cap, ws_bytes, 256), dtype=torch.uint8, device=dev)
                workspace._xkb200_scratch = ws
        else:
            sorted_ids = torch.empty(max_pad, dtype=torch.int32, device=dev)
            expert_ids = torch.empty(max(max_blocks, 1), dtype=torch.int32, device=dev)
            num_post = torch.empty(1, dtype=torch.int32, device=dev)
            if max_blocks == 0:
                expert_ids.zero_()
            # up to 8192 slots the sort takes no scratch memory (new_empty: half the host time of torch.empty)
            ws = ids.new_empty(-(-ws_bytes // 4)) if numel > 8192 else None
        _lib.check(
            lib.xkb_moe_align_block_size(
                _ptr(ids), numel, num_experts, block_size, _ptr(emap),
                0 if emap is None else emap.numel(), _ptr(sorted_ids), _ptr(expert_ids),
                _ptr(num_post), 0, _ptr(ws), 0 if ws is None else ws.numel() * ws.element_size(), _stream(dev)),
            "xkb_moe_align_block_size")
    if sorted_ids.numel() != max_pad:
        sorted_ids = sorted_ids[:max_pad]
    if truncate:
        used = int(num_post.item()) // block_size
        expert_ids = expert_ids[: max(used, 1)]
    elif expert_ids.numel() != max(max_blocks, 1):
        expert_ids = expert_ids[: max(max_blocks, 1)]
    return sorted_ids, expert_ids, num_post


# ---------------------------------------------------------------------------
_LOGIT_DT = {torch.bfloat16: _lib.XKB_BF16, torch.float32: _lib.XKB_F32, torch.float16: _lib.XKB_F16}


def topk_softmax(gating_output, topk, renormalize=True):
    """MoE router: fp32 softmax over all experts, top-k in descending probability (ties: ascending
    expert id), optional renormalisation.  Returns ``(topk_weights [M, topk] fp32, topk_ids [M, topk]
    int32)``.

    Reference: ``topk_softmax_ref`` (src/xkernels/ops/moe/topk_softmax.py:33-95).
    """
    got = (_lib._calls or _lib.load_calls()).topk_softmax(gating_output, topk, renormalize)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_topk_softmax")
        return got
    lib = _lib.load()
    dev = _require_cuda("topk_softmax", gating_output)
    if gating_output.dim() != 2:
        raise ValueError("gating_output must be [M, E]")
    if gating_output.dtype not in _LOGIT_DT:
        raise TypeError(f"topk_softmax: logits must be bf16, fp16 or fp32, got {gating_output.dtype}")
    M, E = gating_output.shape
    if not (1 <= int(topk) <= E):
        raise ValueError(f"topk must satisfy 1 <= topk <= E (got topk={topk}, E={E})")
    g = gating_output.contiguous()
    with _on(dev):
        w = torch.empty((M, int(topk)), dtype=torch.float32, device=dev)
        ids = torch.empty((M, int(topk)), dtype=torch.int32, device=dev)
        _lib.check(
            lib.xkb_topk_softmax(_ptr(g), _LOGIT_DT[g.dtype], _ptr(w), _ptr(ids), M, E, int(topk),
                                 1 if renormalize else 0, _stream(dev)),
            "xkb_topk_softmax")
    return w, ids


# ---------------------------------------------------------------------------
def moe_sum_reduce(y, w=None, routed_scaling_factor=1.0):
    """``out[m] = routed_scaling_factor * sum_k w[m,k] * y[m,k,:]`` in fp32, ascending k.

    Reference: ``moe_sum_reduce_ref`` (src/xkernels/ops/moe/sum_reduce.py:20-39).
    ``y`` is ``[M, top_k, H]`` bf16/fp32, ``w`` ``[M, top_k]`` fp32/bf16 or None;
    the result has ``y.dtype``.
    """
    got = (_lib._calls or _lib.load_calls()).moe_sum_reduce(y, w, routed_scaling_factor)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_moe_sum_reduce")
        return got
    lib = _lib.load()
    dev = _require_cuda("moe_sum_reduce", y, w)
    if y.dim() != 3:
        raise ValueError("y must be [M, top_k, H]")
    if y.dtype not in _DT:
        raise TypeError(f"moe_sum_reduce: unsupported y dtype {y.dtype}")
    y = y.contiguous()
    M, top_k, H = y.shape
    if w is not None:
        if w.dtype not in _DT:
            w = w.to(torch.float32)
        if tuple(w.shape) != (M, top_k):
            raise ValueError(f"w must be [M, top_k] = [{M}, {top_k}], got {tuple(w.shape)}")
        w = w.contiguous()
    with _on(dev):
        out = torch.empty((M, H), dtype=y.dtype, device=dev)
        _lib.check(
            lib.xkb_moe_sum_reduce(_ptr(y), _DT[y.dtype], _ptr(w),
                                   _lib.XKB_F32 if w is None else _DT[w.dtype], _ptr(out),
                                   _DT[y.dtype], M, top_k, H, float(routed_scaling_factor),
                                   _stream(dev)),
            "xkb_moe_sum_reduce")
    return out


def _typed(name, what, t, shape, dtype):
    """``t`` as a contiguous tensor of ``dtype``, after a look at its shape."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name}: {what} must be {list(shape)}, got {list(t.shape)}")
    return (t if t.dtype == dtype else t.to(dtype)).contiguous()


def _mask(name, token_mask, M):
    if token_mask is None:
        return None
    if token_mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"{name}: token_mask must be bool or uint8, got {token_mask.dtype}")
    if tuple(token_mask.shape) != (M,):
        raise ValueError(f"{name}: token_mask must be [{M}], got {list(token_mask.shape)}")
    return token_mask.contiguous()


def _gating(name, gating_output, topk_ids):
    if gating_output.dim() != 2:
        raise ValueError(f"{name}: gating_output must be [M, E]")
    if gating_output.dtype not in _LOGIT_DT:
        raise TypeError(f"{name}: logits must be bf16, fp16 or fp32, got {gating_output.dtype}")
    M, E = gating_output.shape
    if E < 1:
        raise ValueError(f"{name}: no experts")
    if topk_ids is not None:
        if topk_ids.dim() != 2 or topk_ids.shape[0] != M:
            raise ValueError(f"{name}: topk_ids must be [{M}, top_k], got {list(topk_ids.shape)}")
        if topk_ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: topk_ids must be int32 or int64, got {topk_ids.dtype}")
        if topk_ids.dtype == torch.int64:       # what no int32 holds stays outside [0, E)
            topk_ids = topk_ids.clamp(-1, E)
        topk_ids = topk_ids.to(torch.int32).contiguous()
    return gating_output.contiguous(), topk_ids, M, E


def moe_sum_reduce_backward(grad_out, y, w=None, routed_scaling_factor=1.0, need_grad_y=True, need_grad_w=True):
    """The gradients of :func:`moe_sum_reduce`: ``(grad_y, grad_w)``, of ``y``'s and ``w``'s shape and dtype.

    ``grad_y[m,k] = f * w[m,k] * grad_out[m]`` and ``grad_w[m,k] = f * sum_h grad_out[m,h] * y[m,k,h]``, sums in fp32 in a fixed
    order.  What is not wanted, and ``grad_w`` without ``w``, is None.  No reference counterpart: the reference's
    pure-torch form is differentiated by torch.
    """
    got = (_lib._calls or _lib.load_calls()).moe_sum_reduce_backward(grad_out, y, w, routed_scaling_factor, need_grad_y, need_grad_w)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_moe_sum_reduce_backward")
        return got
    lib = _lib.load()
    dev = _require_cuda("moe_sum_reduce_backward", grad_out, y, w)
    if y.dim() != 3:
        raise ValueError("y must be [M, top_k, H]")
    if y.dtype not in _DT:
        raise TypeError(f"moe_sum_reduce_backward: unsupported y dtype {y.dtype}")
    M, top_k, H = y.shape
    grad_out = _typed("moe_sum_reduce_backward", "grad_out", grad_out, (M, H), y.dtype)
    need_grad_w = need_grad_w and w is not None
    w_as = None
    if w is not None:
        w_as = _typed("moe_sum_reduce_backward", "w", w, (M, top_k), w.dtype if w.dtype in _DT else torch.float32)
    if need_grad_w:
        y = y.contiguous()
    with _on(dev):
        grad_y = torch.empty((M, top_k, H), dtype=y.dtype, device=dev) if need_grad_y else None
        grad_w = torch.empty((M, top_k), dtype=w_as.dtype, device=dev) if need_grad_w else None
        _lib.check(
            lib.xkb_moe_sum_reduce_backward(
                _ptr(grad_out), _DT[y.dtype], _ptr(y) if need_grad_w else 0, _ptr(w_as),
                _lib.XKB_F32 if w_as is None else _DT[w_as.dtype], _ptr(grad_y), _ptr(grad_w), M, top_k, H,
                float(routed_scaling_factor), _stream(dev)),
            "xkb_moe_sum_reduce_backward")
    if grad_w is not None and grad_w.dtype != w.dtype:
        grad_w = grad_w.to(w.dtype)
    return grad_y, grad_w


class BalanceLoss(NamedTuple):
    """What :func:`moe_balance_loss` returns."""

    loss: torch.Tensor         # [] fp32
    counts: torch.Tensor       # [E] int32: slots per expert
    mean_probs: torch.Tensor   # [E] fp32: mean router probability per expert
    tokens: torch.Tensor       # [] int32: tokens that count


def moe_balance_loss(gating_output, topk_ids, token_mask=None):
    """Balance loss and per-expert counts of a routing: ``E * sum_e counts[e] / (top_k * T) * mean_probs[e]``, which is 1
    for an even one.

    ``gating_output`` ``[M, E]`` logits as for :func:`topk_softmax`, ``topk_ids`` ``[M, top_k]`` its choice (ids outside
    ``[0, E)`` are dropped slots: not counted), ``token_mask`` ``[M]`` bool: padding tokens (False) count for nothing; ``T`` is the
    number of the others.  Without one (``T = 0``) the loss is 0.  A row of logits that are all -inf adds nothing to ``mean_probs``.
    The same bits in every run.  The gradient: :func:`moe_router_backward`; in a data-parallel job ``counts`` and ``tokens`` may be
    summed over the ranks before it, which makes it the gradient of the whole batch's loss.  No reference counterpart.
    """
    got = (_lib._calls or _lib.load_calls()).moe_balance_loss(gating_output, topk_ids, token_mask)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_moe_balance_loss")
        return BalanceLoss._make(got)
    lib = _lib.load()
    dev = _require_cuda("moe_balance_loss", gating_output, topk_ids, token_mask)
    if topk_ids is None:
        raise TypeError("moe_balance_loss: topk_ids is missing")
    g, ids, M, E = _gating("moe_balance_loss", gating_output, topk_ids)
    mask = _mask("moe_balance_loss", token_mask, M)
    with _on(dev):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        counts = torch.empty((E,), dtype=torch.int32, device=dev)
        mean = torch.empty((E,), dtype=torch.float32, device=dev)
        tokens = torch.empty((), dtype=torch.int32, device=dev)
        ws_bytes = max(_bytes("xkb_moe_balance_loss_workspace_bytes", M, E), 0)   # of this call alone: calls may overlap
        ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
        _lib.check(
            lib.xkb_moe_balance_loss(_ptr(g), _LOGIT_DT[g.dtype], _ptr(ids), _ptr(mask), _ptr(loss), _ptr(counts),
                                     _ptr(mean), _ptr(tokens), M, E, ids.shape[1], _ptr(ws), ws_bytes, _stream(dev)),
            "xkb_moe_balance_loss")
    return BalanceLoss(loss, counts, mean, tokens)


def moe_router_backward(gating_output, topk_ids, grad_weights=None, renormalize=True, counts=None, tokens=None,
                        grad_loss=None, token_mask=None):
    """The gradient of the gating logits, ``[M, E]`` of their dtype, in one pass.

    From the routing weights: ``grad_weights`` ``[M, top_k]``, the gradient of :func:`topk_softmax`'s weights for
    ``topk_ids`` (``renormalize`` as there).  Ids outside ``[0, E)`` are dropped slots, and renormalised weights are taken to be
    ``p_j`` by the sum over the other slots.  A caller that drops slots behind :func:`topk_softmax`, which divided by the sum over all of
    them, therefore passes the ids as they were, and a gradient of 0 for what was dropped.  From :func:`moe_balance_loss`: ``counts`` and
    ``tokens`` (None: M) as it returned them, ``grad_loss`` the loss's gradient (a number or a one-element CUDA tensor; None: 1),
    ``token_mask`` as there.  Either may be left out.  A row that neither brings a gradient to is 0, whatever its logits.  No
    reference counterpart: the reference's pure-torch router is differentiated by torch.
    """
    got = (_lib._calls or _lib.load_calls()).moe_router_backward(
        gating_output, topk_ids, grad_weights, renormalize, counts, tokens, grad_loss, token_mask)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_moe_router_backward")
        return got
    lib = _lib.load()
    name = "moe_router_backward"
    on_device = grad_loss if isinstance(grad_loss, torch.Tensor) else None
    dev = _require_cuda(name, gating_output, topk_ids, grad_weights, counts, tokens, on_device, token_mask)
    if grad_weights is None and counts is None:
        raise ValueError(f"{name}: neither grad_weights nor counts")
    if counts is None and (grad_loss is not None or tokens is not None):
        raise ValueError(f"{name}: grad_loss and tokens belong to counts")
    if topk_ids is None:
        raise TypeError(f"{name}: topk_ids is missing")
    g, ids, M, E = _gating(name, gating_output, topk_ids)
    top_k = ids.shape[1]
    mask = _mask(name, token_mask, M)
    gw = None if grad_weights is None else _typed(name, "grad_weights", grad_weights, (M, top_k), torch.float32)
    scale = 1.0
    if counts is not None:
        counts = _typed(name, "counts", counts, (E,), torch.int32)
        if tokens is not None:
            tokens = _typed(name, "tokens", tokens.reshape(-1), (1,), torch.int32)
        if on_device is not None:
            on_device = _typed(name, "grad_loss", on_device.reshape(-1), (1,), torch.float32)
        elif grad_loss is not None:
            scale = float(grad_loss)
    with _on(dev):
        out = torch.empty((M, E), dtype=g.dtype, device=dev)
        _lib.check(
            lib.xkb_moe_router_backward(_ptr(g), _LOGIT_DT[g.dtype], _ptr(ids), _ptr(gw), 1 if renormalize else 0,
                                        _ptr(counts), _ptr(tokens), _ptr(on_device), scale, _ptr(mask), _ptr(out), M, E,
                                        top_k, _stream(dev)),
            "xkb_moe_router_backward")
    return out


# ---------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns."""

    logprobs: torch.Tensor       # [M] fp32
    entropy: torch.Tensor        # [M] fp32, nats
    stats: torch.Tensor          # [M, 2] fp32: row maximum m, ln sum exp(x - m)
    top_logprobs: torch.Tensor   # [M, top_k] fp32, descending
    top_ids: torch.Tensor        # [M, top_k] int32


def _head(name, logits, token_ids):
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{name}: logits must be [M, V]")
    if logits.dtype not in _LOGIT_DT:
        raise TypeError(f"{name}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    M, V = logits.shape
    if token_ids is not None:
        if token_ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: token_ids must be int32 or int64, got {token_ids.dtype}")
        if tuple(token_ids.shape) != (M,):
            raise ValueError(f"{name}: token_ids must be [{M}], got {list(token_ids.shape)}")
        token_ids = token_ids.contiguous()
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    return logits, token_ids, M, V


def token_logprobs(logits, token_ids, top_k=0):
    """Log-probabilities of given tokens, entropy, and the ``top_k`` likeliest tokens of every row of a head's logits.

    ``logits`` ``[M, V]`` bf16, fp16 or fp32; rows may lie apart (a slice of a padded head is read in place).  ``token_ids``
    ``[M]`` int32 or int64; a negative id is padding and has log-probability 0, an id of V or more gives NaN.  ``top_k`` up to
    ``min(V, 64)``; alternatives come in descending probability, ties by ascending id as in :func:`topk_softmax`.  A row whose
    logits are all -inf has log-probabilities -inf and entropy 0, a row with a NaN or a +inf is NaN.  The same bits in every
    run.  The gradient: :func:`token_logprobs_backward`.  No reference counterpart.
    """
    got = (_lib._calls or _lib.load_calls()).token_logprobs(logits, token_ids, top_k)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_token_logprobs")
        return TokenLogprobs._make(got)
    lib = _lib.load()
    name = "token_logprobs"
    dev = _require_cuda(name, logits, token_ids)
    if token_ids is None:
        raise TypeError(f"{name}: token_ids is missing")
    logits, ids, M, V = _head(name, logits, token_ids)
    top_k = int(top_k)
    if not 0 <= top_k <= min(V, 64):
        raise ValueError(f"{name}: top_k must satisfy 0 <= top_k <= min(V, 64) (got top_k={top_k}, V={V})")
    with _on(dev):
        lp = torch.empty((M,), dtype=torch.float32, device=dev)
        entropy = torch.empty((M,), dtype=torch.float32, device=dev)
        stats = torch.empty((M, 2), dtype=torch.float32, device=dev)
        top_lp = torch.empty((M, top_k), dtype=torch.float32, device=dev)
        top_ids = torch.empty((M, top_k), dtype=torch.int32, device=dev)
        _lib.check(
            lib.xkb_token_logprobs(_ptr(logits), _LOGIT_DT[logits.dtype], logits.stride(0), _ptr(ids),
                                   1 if ids.dtype == torch.int64 else 0, _ptr(lp), _ptr(entropy), _ptr(stats),
                                   _ptr(top_lp), _ptr(top_ids), M, V, top_k, _stream(dev)),
            "xkb_token_logprobs")
    return TokenLogprobs(lp, entropy, stats, top_lp, top_ids)


def token_logprobs_backward(logits, token_ids, stats, entropy=None, grad_logprobs=None, grad_entropy=None, top_ids=None,
                            grad_top_logprobs=None):
    """The gradient of a head's logits, ``[M, V]`` of their dtype, from those of :func:`token_logprobs`'s outputs.

    ``stats``, ``entropy`` (for ``grad_entropy``) and ``top_ids`` (for ``grad_top_logprobs``) are what the forward call returned.
    Gradients that are left out count as 0; one at least is needed.  Padding tokens (negative ids) have no gradient.  The
    result is contiguous, or, where the logits' rows do not start on 16 bytes, a view of rows that start like theirs.
    """
    got = (_lib._calls or _lib.load_calls()).token_logprobs_backward(
        logits, token_ids, stats, entropy, grad_logprobs, grad_entropy, top_ids, grad_top_logprobs)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_token_logprobs_backward")
        return got
    lib = _lib.load()
    name = "token_logprobs_backward"
    dev = _require_cuda(name, logits, token_ids, stats, entropy, grad_logprobs, grad_entropy, top_ids, grad_top_logprobs)
    if grad_logprobs is None and grad_entropy is None and grad_top_logprobs is None:
        raise ValueError(f"{name}: no gradient is given")
    if (grad_logprobs is not None and token_ids is None) or (grad_entropy is not None and entropy is None) or \
            (grad_top_logprobs is not None and top_ids is None):
        raise ValueError(f"{name}: grad_logprobs needs token_ids, grad_entropy needs entropy, grad_top_logprobs needs top_ids")
    logits, ids, M, V = _head(name, logits, token_ids)
    stats = _typed(name, "stats", stats, (M, 2), torch.float32)
    if grad_logprobs is not None:
        grad_logprobs = _typed(name, "grad_logprobs", grad_logprobs, (M,), torch.float32)
    if grad_entropy is not None:
        grad_entropy = _typed(name, "grad_entropy", grad_entropy, (M,), torch.float32)
        entropy = _typed(name, "entropy", entropy, (M,), torch.float32)
    top_k = 0
    if grad_top_logprobs is not None:
        top_k = int(top_ids.shape[-1]) if top_ids.dim() else 0
        if top_ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: top_ids must be int32 or int64, got {top_ids.dtype}")
        if top_ids.dtype == torch.int64:
            top_ids = top_ids.clamp(-1, V)
        top_ids = _typed(name, "top_ids", top_ids, (M, top_k), torch.int32)
        grad_top_logprobs = _typed(name, "grad_top_logprobs", grad_top_logprobs, (M, top_k), torch.float32)
        if top_k > 64:
            raise ValueError(f"{name}: at most 64 alternatives (got {top_k})")
    # rows of the gradient start where rows of the logits do within 16 bytes, so that both go in 16-byte pieces
    es = logits.element_size()
    ld, shift = logits.stride(0), logits.data_ptr() % 16 // es
    ld_grad = V if M <= 1 else V + (ld - V) % (16 // es)
    with _on(dev):
        if ld_grad == V and shift == 0:
            out = torch.empty((M, V), dtype=logits.dtype, device=dev)
        else:
            out = torch.empty((M * ld_grad + shift,), dtype=logits.dtype, device=dev).as_strided((M, V), (ld_grad, 1), shift)
        _lib.check(
            lib.xkb_token_logprobs_backward(
                _ptr(logits), _LOGIT_DT[logits.dtype], ld, _ptr(ids), 1 if ids is not None and ids.dtype == torch.int64 else 0,
                _ptr(stats), _ptr(entropy) if grad_entropy is not None else 0, _ptr(grad_logprobs), _ptr(grad_entropy),
                _ptr(top_ids) if top_k else 0, _ptr(grad_top_logprobs) if top_k else 0, top_k, _ptr(out), ld_grad, M, V,
                _stream(dev)),
            "xkb_token_logprobs_backward")
    return out


# ---------------------------------------------------------------------------
_HALF_DT = {torch.bfloat16: _lib.XKB_BF16, torch.float16: _lib.XKB_F16}


def _given(name, **tensors) -> None:
    for what, t in tensors.items():
        if t is None:
            raise TypeError(f"{name}: {what} is missing")


def _matrix(name, what, t, shape, dtype):
    """``t`` as an operand of a dense product: of ``dtype``, rows a multiple of 16 bytes apart, the first on 16 bytes.  Read in
    place where it is one already (a slice of wider rows too); else laid out once more."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name}: {what} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: {what} must be {dtype} like the first argument, got {t.dtype}")
    rows, cols = shape
    if (cols == 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(0) >= cols:
        return t, t.stride(0)
    ld = -(-cols // 8) * 8
    buf = torch.empty((rows, ld), dtype=dtype, device=t.device)
    buf[:, :cols].copy_(t)
    return buf, ld


class LinearCrossEntropy(NamedTuple):
    """What :func:`linear_cross_entropy` returns."""

    loss: torch.Tensor    # [M] fp32
    lse: torch.Tensor     # [M] fp32: log-sum-exp of the logits
    stats: torch.Tensor   # [M, 2] fp32: row maximum m, ln sum exp(z - m)


def _linear_head(name, hidden, weight, labels):
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{name}: hidden must be [M, H] and weight [V, H]")
    if hidden.dtype not in _HALF_DT:
        raise TypeError(f"{name}: hidden must be bf16 or fp16, got {hidden.dtype}")
    if labels.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: labels must be int32 or int64, got {labels.dtype}")
    M, H = hidden.shape
    if tuple(labels.shape) != (M,):
        raise ValueError(f"{name}: labels must be [{M}], got {list(labels.shape)}")
    if H > 1 and hidden.stride(1) != 1:
        hidden = hidden.contiguous()
    return hidden, labels.contiguous(), M, H, weight.shape[0]


def linear_cross_entropy(hidden, weight, labels):
    """Cross entropy of a head: ``loss[i] = lse(z[i]) - z[i, labels[i]]`` with ``z = hidden @ weight.T``, which is never stored.

    ``hidden`` ``[M, H]`` and ``weight`` ``[V, H]`` bf16 or fp16 (products are added up in fp32), ``labels`` ``[M]`` int32 or int64.
    A negative label is padding: its results are 0, and what the row holds has no influence on any other.  Among more than 128 rows it
    is not read and costs next to nothing; up to 128 are multiplied together, which takes as long whatever they are.  A label of V or
    more gives a loss of NaN, a row whose logits hold a NaN or +inf is NaN.  The same bits in every run.  Where :func:`token_logprobs` takes
    logits, this takes what they are made from; its gradient is :func:`linear_cross_entropy_backward`.  No reference counterpart.
    """
    got = (_lib._calls or _lib.load_calls()).linear_cross_entropy(hidden, weight, labels)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_linear_cross_entropy")
        return LinearCrossEntropy._make(got)
    lib = _lib.load()
    name = "linear_cross_entropy"
    _given(name, hidden=hidden, weight=weight, labels=labels)
    dev = _require_cuda(name, hidden, weight, labels)
    hidden, labels, M, H, V = _linear_head(name, hidden, weight, labels)
    with _on(dev):
        weight, ld_w = _matrix(name, "weight", weight, (V, H), hidden.dtype)
        loss = torch.empty((M,), dtype=torch.float32, device=dev)
        lse = torch.empty((M,), dtype=torch.float32, device=dev)
        stats = torch.empty((M, 2), dtype=torch.float32, device=dev)
        ws_bytes = _bytes("xkb_linear_cross_entropy_workspace_bytes", M, H, V)      # of this call alone: calls may overlap
        ws = torch.empty((max(ws_bytes, 0),), dtype=torch.uint8, device=dev)
        _lib.check(
            lib.xkb_linear_cross_entropy(_ptr(hidden), hidden.stride(0), _HALF_DT[hidden.dtype], _ptr(weight), ld_w, _ptr(labels),
                                         1 if labels.dtype == torch.int64 else 0, _ptr(loss), _ptr(lse), _ptr(stats), M, H, V,
                                         _ptr(ws), ws_bytes, _stream(dev)),
            "xkb_linear_cross_entropy")
    return LinearCrossEntropy(loss, lse, stats)


def linear_cross_entropy_backward(hidden, weight, labels, stats, grad_loss=None, grad_lse=None, need_grad_hidden=True,
                                  need_grad_weight=True):
    """The gradients of :func:`linear_cross_entropy`: ``(grad_hidden, grad_weight)``, of ``hidden``'s and ``weight``'s shape and
    dtype; what is not wanted is None.

    ``stats`` is what the forward call returned; ``grad_loss`` and ``grad_lse`` ``[M]`` are the gradients of its outputs (one at
    least is needed; the other counts as 0; of padding rows they are not read).  The logits are multiplied once more, a piece of the
    vocabulary at a time, so 256 MiB of their gradient are held at most (or 256 columns of it, which is more beyond 2^19 rows), besides
    a copy of the rows and, where there are several pieces or sums go in parts, fp32 sums of ``grad_hidden``.  Sums are fp32; the
    gradient of the logits is rounded to ``hidden``'s dtype (up to 16 rows: held in two terms of it) as the operand of the next
    products.  The same bits in every run.
    """
    got = (_lib._calls or _lib.load_calls()).linear_cross_entropy_backward(
        hidden, weight, labels, stats, grad_loss, grad_lse, need_grad_hidden, need_grad_weight)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_linear_cross_entropy_backward")
        return got
    lib = _lib.load()
    name = "linear_cross_entropy_backward"
    _given(name, hidden=hidden, weight=weight, labels=labels, stats=stats)
    dev = _require_cuda(name, hidden, weight, labels, stats, grad_loss, grad_lse)
    if grad_loss is None and grad_lse is None:
        raise ValueError(f"{name}: no gradient is given")
    hidden, labels, M, H, V = _linear_head(name, hidden, weight, labels)
    stats = _typed(name, "stats", stats, (M, 2), torch.float32)
    if grad_loss is not None:
        grad_loss = _typed(name, "grad_loss", grad_loss, (M,), torch.float32)
    if grad_lse is not None:
        grad_lse = _typed(name, "grad_lse", grad_lse, (M,), torch.float32)
    with _on(dev):
        weight, ld_w = _matrix(name, "weight", weight, (V, H), hidden.dtype)
        grad_hidden = torch.empty((M, H), dtype=hidden.dtype, device=dev) if need_grad_hidden else None
        grad_weight = torch.empty((V, H), dtype=hidden.dtype, device=dev) if need_grad_weight else None
        ws_bytes = _bytes("xkb_linear_cross_entropy_backward_workspace_bytes", M, H, V)
        ws = torch.empty((max(ws_bytes, 0),), dtype=torch.uint8, device=dev)
        _lib.check(
            lib.xkb_linear_cross_entropy_backward(
                _ptr(hidden), hidden.stride(0), _HALF_DT[hidden.dtype], _ptr(weight), ld_w, _ptr(labels), 1 if labels.dtype == torch.int64 else 0,
                _ptr(stats), _ptr(grad_loss), _ptr(grad_lse), _ptr(grad_hidden), _ptr(grad_weight), M, H, V, _ptr(ws), ws_bytes,
                _stream(dev)),
            "xkb_linear_cross_entropy_backward")
    return grad_hidden, grad_weight


def _gated_sizes(name, x, w13, w2):
    if x.dim() != 2 or w13.dim() != 2 or w2.dim() != 2:
        raise ValueError(f"{name}: x must be [M, H], w13 [2*I, H] and w2 [H, I]")
    if x.dtype not in _HALF_DT:
        raise TypeError(f"{name}: x must be bf16 or fp16, got {x.dtype}")
    (M, H), I = x.shape, w2.shape[1]
    if H < 1 or I < 1:
        raise ValueError(f"{name}: empty weights")
    return M, H, I


def gated_ffn(x, w13, w2, swiglu_limit=None, save_gate_up=False):
    """A dense gated feed-forward block, such as the shared expert beside the routed ones: ``(silu(gate) * up) @ w2.T`` with
    ``gate, up = x @ w13.T``.

    ``x`` ``[M, H]``, ``w13`` ``[2*I, H]`` (gate rows first, as in :func:`fused_moe_mxfp4`), ``w2`` ``[H, I]``, all bf16 or all fp16;
    rows may lie apart.  ``swiglu_limit`` (None or 0: none) cuts gate off at the limit and up at plus and minus it, as there.
    Products are added up in fp32, and ``silu(gate) * up`` is rounded to ``x``'s dtype once, as the operand of the second product (up to
    16 rows: held in two terms of it); beyond fp16's 65504 it is infinite.
    Returns ``out`` ``[M, H]``, or ``(out, gate_up)`` with ``save_gate_up``: ``[M, 2*I]`` before the limit, for
    :func:`gated_ffn_backward`.  The same bits in every run.  No reference counterpart.
    """
    got = (_lib._calls or _lib.load_calls()).gated_ffn(x, w13, w2, swiglu_limit, save_gate_up)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_gated_ffn")
        return got
    lib = _lib.load()
    name = "gated_ffn"
    _given(name, x=x, w13=w13, w2=w2)
    dev = _require_cuda(name, x, w13, w2)
    M, H, I = _gated_sizes(name, x, w13, w2)
    limit = 0.0 if swiglu_limit is None else float(swiglu_limit)
    with _on(dev):
        dt = x.dtype
        x, ld_x = _matrix(name, "x", x, (M, H), dt)
        w13, ld_13 = _matrix(name, "w13", w13, (2 * I, H), dt)
        w2, ld_2 = _matrix(name, "w2", w2, (H, I), dt)
        out = torch.empty((M, H), dtype=dt, device=dev)
        gate_up = torch.empty((M, 2 * I), dtype=dt, device=dev) if save_gate_up else None
        ws_bytes = _bytes("xkb_gated_ffn_workspace_bytes", M, H, I)                 # of this call alone: calls may overlap
        ws = torch.empty((max(ws_bytes, 0),), dtype=torch.uint8, device=dev)
        _lib.check(
            lib.xkb_gated_ffn(_ptr(x), ld_x, _HALF_DT[dt], _ptr(w13), ld_13, _ptr(w2), ld_2, limit, _ptr(out), _ptr(gate_up), M, H, I,
                              _ptr(ws), ws_bytes, _stream(dev)),
            "xkb_gated_ffn")
    return (out, gate_up) if save_gate_up else out


def gated_ffn_backward(grad_out, x, w13, w2, gate_up=None, swiglu_limit=None, need_grad_x=True, need_grad_w13=True,
                       need_grad_w2=True):
    """The gradients of :func:`gated_ffn`: ``(grad_x, grad_w13, grad_w2)``, of their shapes and dtype; what is not wanted is None.

    ``gate_up`` is what the forward call saved; without it the first product is multiplied once more (and what the limit cuts off is
    then decided on its result rounded to ``x``'s dtype, as with the saved one).  Gradients of gate and up and ``silu(gate) * up`` are
    rounded to ``x``'s dtype once, as operands of the next products (up to 16 rows: held in two terms of it), and not scaled: in fp16 scale
    the loss, for below 6e-5 they lose bits.  All sums are fp32.  The same bits in every run.
    """
    got = (_lib._calls or _lib.load_calls()).gated_ffn_backward(
        grad_out, x, w13, w2, gate_up, swiglu_limit, need_grad_x, need_grad_w13, need_grad_w2)
    if got is not None:
        if type(got) is int:
            _lib.check(got, "xkb_gated_ffn_backward")
        return got
    lib = _lib.load()
    name = "gated_ffn_backward"
    _given(name, grad_out=grad_out, x=x, w13=w13, w2=w2)
    dev = _require_cuda(name, grad_out, x, w13, w2, gate_up)
    M, H, I = _gated_sizes(name, x, w13, w2)
    limit = 0.0 if swiglu_limit is None else float(swiglu_limit)
    dt = x.dtype
    if gate_up is not None:
        if gate_up.dtype != dt:
            raise TypeError(f"{name}: gate_up must be {dt} like x, got {gate_up.dtype}")
        gate_up = _typed(name, "gate_up", gate_up, (M, 2 * I), dt)
    with _on(dev):
        grad_out, ld_go = _matrix(name, "grad_out", grad_out, (M, H), dt)
        x, ld_x = _matrix(name, "x", x, (M, H), dt)
        w13, ld_13 = _matrix(name, "w13", w13, (2 * I, H), dt)
        w2, ld_2 = _matrix(name, "w2", w2, (H, I), dt)
        grad_x = torch.empty((M, H), dtype=dt, device=dev) if need_grad_x else None
        grad_w13 = torch.empty((2 * I, H), dtype=dt, device=dev) if need_grad_w13 else None
        grad_w2 = torch.empty((H, I), dtype=dt, device=dev) if need_grad_w2 else None
        ws_bytes = _bytes("xkb_gated_ffn_backward_workspace_bytes", M, H, I, 0 if gate_up is not None else 1)
        ws = torch.empty((max(ws_bytes, 0),), dtype=torch.uint8, device=dev)
        _lib.check(
            lib.xkb_gated_ffn_backward(
                _ptr(grad_out), ld_go, _HALF_DT[dt], _ptr(x), ld_x, _ptr(w13), ld_13, _ptr(w2), ld_2, _ptr(gate_up), limit, _ptr(grad_x),
                _ptr(grad_w13), _ptr(grad_w2), M, H, I, _ptr(ws), ws_bytes, _stream(dev)),
            "xkb_gated_ffn_backward")
    return grad_x, grad_w13, grad_w2


# ---------------------------------------------------------------------------
_checked_scales: dict[tuple[int, int], int] = {}
_INT4_SCALE_LIMIT = float(2 ** 24)


def _check_int4_scales(scale: torch.Tensor) -> None:
    """The tcgen05 INT4 dequantiser of groups of 32 is exact for scales below 2^24 in magnitude (it multiplies
    by s * 2^103 in bf16); a larger or non-finite scale would come out as inf/NaN, so such a tensor
    is refused (at every group size: the wider groups' kernels would take it).  Checked once per tensor (keyed by storage address, size and version counter): one
    reduction and one host read on the first call with it, so make that call before a stream capture."""
    key = (scale.data_ptr(), scale.numel())
    if _checked_scales.get(key) == scale._version:
        return
    top = float(scale.abs().max()) if scale.numel() else 0.0
    if not (top < _INT4_SCALE_LIMIT):        # also catches NaN
        raise ValueError(f"fused_moe_int4_w4a16: group scales must be finite and below 2^24 in magnitude (max |scale| = {top})")
    if len(_checked_scales) > 256:
        _checked_scales.clear()
    _checked_scales[key] = scale._version


def _routing_args(name, topk_ids, topk_w, expert_map, dev, M):
    if topk_ids.dim() != 2 or topk_ids.shape[0] != M:
        raise ValueError(f"{name}: topk_ids must be [M, top_k]")
    ids = topk_ids if topk_ids.dtype == torch.int32 else topk_ids.to(torch.int32)
    ids = ids.contiguous()
    tw = topk_w if topk_w.dtype == torch.float32 else topk_w.to(torch.float32)
    tw = tw.contiguous()
    if tuple(tw.shape) != tuple(ids.shape):
        raise ValueError(f"{name}: topk_w shape {tuple(tw.shape)} != topk_ids shape {tuple(ids.shape)}")
    emap = None
    if expert_map is not None:
        emap = expert_map.to(device=dev, dtype=torch.int32).contiguous()
    return ids, tw, emap


def fused_moe_int4_w4a16(A, packed, scale, topk_ids, topk_w, group_size=32, mul_routed_weight=True,
                         fused_combine=None, expert_map=None, workspace=None, *, path="auto"):
    """INT4 W4A16 grouped fused-MoE GEMM ``out[m] = sum_j w[m,j] * (A[m] @ W[e_mj]^T)``.

    Signature of the reference backends (src/xkernels/ops/moe/reference.py:22-33,
    triton/moe_int4_kernel.py:438-449).  ``fused_combine`` is accepted for API
    parity: the combine is always the fixed-order fp32 reduce.  ``workspace``:
    None (this package's per-device buffer), a CUDA uint8 tensor, or the
    reference's ``MoeInt4Workspace`` (see :func:`_caller_workspace`): with the
    latter two every call runs at the same addresses, e.g. under a CUDA graph.
    The tcgen05 kernels never wait without a limit; after a call
    :func:`check_status` (or :func:`check_workspace_status`) tells whether one gave up.
    ``expert_map`` selects the replicated expert-parallel mode (partial output).
    ``path``: ``"auto"`` | ``"simt"`` | ``"tc"``.
    """
    lib = _lib.load()
    dev = _require_cuda("fused_moe_int4_w4a16", A, packed, scale, topk_ids, topk_w, expert_map)
    if A.dtype not in _DT:
        raise TypeError(f"fused_moe_int4_w4a16: A must be bf16 or fp32, got {A.dtype}")
    if packed.dtype != torch.int32 or packed.dim() != 3:
        raise TypeError("fused_moe_int4_w4a16: packed must be int32 [E, N, K//8]")
    A = A.contiguous()
    packed = packed.contiguous()
    M, K = A.shape
    E, N, kp = packed.shape
    group_size = int(group_size)
    if kp * 8 != K:
        raise ValueError(f"packed last dim {kp} != K//8 = {K // 8}")
    if scale.dtype != torch.bfloat16:
        scale = scale.to(torch.bfloat16)
    scale = scale.contiguous()
    if tuple(scale.shape) != (E, N, K // group_size):
        raise ValueError(f"scale must be [E, N, K//group_size] = [{E}, {N}, {K // group_size}]")
    ids, tw, emap = _routing_args("fused_moe_int4_w4a16", topk_ids, topk_w, expert_map, dev, M)
    top_k = ids.shape[1]
    pcode = {"auto": _lib.PATH_AUTO, "simt": _lib.PATH_SIMT, "tc": _lib.PATH_TC}[path]
    if path != "simt":
        _check_int4_scales(scale)
    with _on(dev):
        out = torch.empty((M, N), dtype=A.dtype, device=dev)
        ws_bytes = _bytes("xkb_fused_moe_int4_w4a16_workspace_bytes", M, N, K, E, top_k, _DT[A.dtype])
        fits, cap_bytes = False, ws_bytes
        if workspace is not None and hasattr(workspace, "matches"):
            fits = bool(workspace.matches(M, top_k, N, dtype=A.dtype, device=dev))
            if fits:   # capacity of the object = rows of its combine buffer (workspace.py:199-213)
                cap_bytes = _bytes("xkb_fused_moe_int4_w4a16_workspace_bytes", int(workspace.combine_out.shape[0]), N, K, E,
                                                                             top_k, _DT[A.dtype])
        ws = _caller_workspace(workspace, fits, cap_bytes, dev, ws_bytes)
        _lib.check(
            lib.xkb_fused_moe_int4_w4a16(
                _ptr(A), _DT[A.dtype], _ptr(packed), _ptr(scale), _ptr(ids), _ptr(tw), _ptr(emap),
                0 if emap is None else emap.numel(), _ptr(out), M, N, K, E, top_k, group_size,
                1 if mul_routed_weight else 0, pcode, _ptr(ws), ws.numel(), _stream(dev)),
            "xkb_fused_moe_int4_w4a16")
    return out


def fused_moe_mxfp4(A, w13, w13_scale, w2, w2_scale, topk_ids, topk_w, b13=None, b2=None,
                    swiglu_limit=10.0, group_size=32, mul_routed_weight=True, expert_map=None,
                    workspace=None, *, path="auto"):
    """MXFP4 fused MoE: gate_up GEMM -> clamped SwiGLU -> down GEMM -> weighted combine.

    Signature of the reference backends
    (src/xkernels/ops/moe/mxfp4_reference.py:28-43, triton/moe_mxfp4_kernel.py:487-502).
    ``w13`` ``[E, 2*ispp, hidden//2]`` and ``w2`` ``[E, hidden, ispp//2]`` are uint8
    E2M1 pairs, the scales uint8 e8m0 per 32 elements.  The three bf16 rounding
    points of the reference (gate_up, activation, down) are reproduced.
    ``workspace`` as in :func:`fused_moe_int4_w4a16` (None, a CUDA uint8 tensor or the reference's
    ``MoeMxfp4Workspace``).  After a call :func:`check_status` (or :func:`check_workspace_status`)
    reports a kernel that gave up a bounded wait, a scale byte the prefill-sized tcgen05 instance
    does not convert (191..254), or a routing value out of range.
    """
    lib = _lib.load()
    dev = _require_cuda("fused_moe_mxfp4", A, w13, w13_scale, w2, w2_scale, topk_ids, topk_w, b13, b2,
                        expert_map)
    if int(group_size) != 32:
        raise ValueError("fused_moe_mxfp4: the MX block size is 32")
    if A.dtype not in _DT:
        raise TypeError(f"fused_moe_mxfp4: A must be bf16 or fp32, got {A.dtype}")
    for name, t in (("w13", w13), ("w13_scale", w13_scale), ("w2", w2), ("w2_scale", w2_scale)):
        if t.dtype != torch.uint8:
            raise TypeError(f"fused_moe_mxfp4: {name} must be uint8")
    A = A.contiguous()
    w13, w13_scale, w2, w2_scale = (t.contiguous() for t in (w13, w13_scale, w2, w2_scale))
    M, hidden = A.shape
    E, two_ispp, half_hidden = w13.shape
    ispp = two_ispp // 2
    if half_hidden * 2 != hidden or tuple(w2.shape) != (E, hidden, ispp // 2):
        raise ValueError("fused_moe_mxfp4: w13 must be [E, 2*ispp, hidden//2] and w2 [E, hidden, ispp//2]")
    if tuple(w13_scale.shape) != (E, 2 * ispp, hidden // 32) or tuple(w2_scale.shape) != (E, hidden, ispp // 32):
        raise ValueError("fused_moe_mxfp4: scale shapes must be [E,2*ispp,hidden//32] and [E,hidden,ispp//32]")
    if b13 is not None:
        b13 = b13.to(torch.bfloat16).contiguous()
    if b2 is not None:
        b2 = b2.to(torch.bfloat16).contiguous()
    ids, tw, emap = _routing_args("fused_moe_mxfp4", topk_ids, topk_w, expert_map, dev, M)
    top_k = ids.shape[1]
    limit = 0.0 if swiglu_limit is None else float(swiglu_limit)
    pcode = {"auto": _lib.PATH_AUTO, "simt": _lib.PATH_SIMT, "tc": _lib.PATH_TC}[path]
    with _on(dev):
        out = torch.empty((M, hidden), dtype=A.dtype, device=dev)
        ws_bytes = _bytes("xkb_fused_moe_mxfp4_workspace_bytes", M, hidden, ispp, E, top_k)
        fits, cap_bytes = False, ws_bytes
        if workspace is not None and hasattr(workspace, "out") and hasattr(workspace, "act"):
            # matches() of MoeMxfp4Workspace wants the align block of ITS kernel; what matters here is
            # that the object was built for this problem: same ispp / hidden / dtype, enough rows
            fits = (workspace.act.shape[1] == ispp and workspace.out.shape[1] == hidden and workspace.out.shape[0] >= M
                    and workspace.act.dtype == A.dtype and workspace.act.device == dev)
            if fits:
                cap_bytes = _bytes("xkb_fused_moe_mxfp4_workspace_bytes", int(workspace.out.shape[0]), hidden, ispp, E, top_k)
        ws = _caller_workspace(workspace, fits, cap_bytes, dev, ws_bytes)
        _lib.check(
            lib.xkb_fused_moe_mxfp4(
                _ptr(A), _DT[A.dtype], _ptr(w13), _ptr(w13_scale), _ptr(w2), _ptr(w2_scale), _ptr(ids),
                _ptr(tw), _ptr(b13), _ptr(b2), _ptr(emap), 0 if emap is None else emap.numel(),
                _ptr(out), M, hidden, ispp, E, top_k, limit, 1 if mul_routed_weight else 0, pcode,
                _ptr(ws), ws.numel(), _stream(dev)),
            "xkb_fused_moe_mxfp4")
    return out


def fused_moe_int4_ffn(A, w13_packed, w13_scale, w2_packed, w2_scale, topk_ids, topk_w, group_size=32,
                       swiglu_limit=None, expert_map=None, workspace=None, *, path="auto"):
    """One expert layer of two INT4 W4A16 GEMMs in one call: gate_up GEMM -> SwiGLU -> down GEMM ->
    weighted top-k combine.

    The reference has the single GEMM only (``fused_moe_int4_w4a16``, src/xkernels/ops/moe/interface.py:19-32;
    its INT4 benchmark measures the two shapes of such a layer, meta/benchmarks/bench_moe_int4_w4a16.py:3-12).
    This op returns what a caller of the reference gets from composing it: the first GEMM over the
    token's slots (bf16 result), ``act = (silu(gate) * up).to(A.dtype)`` with the gate rows first in
    ``w13``, the second GEMM with the routing weights (bf16 result per slot), ``moe_sum_reduce`` over
    the slots.  ``w13_packed [E, 2*inter, hidden//8]``, ``w13_scale [E, 2*inter, hidden//group]``,
    ``w2_packed [E, hidden, inter//8]``, ``w2_scale [E, hidden, inter//group]``.
    ``workspace`` and :func:`check_status` as in :func:`fused_moe_int4_w4a16`.
    """
    lib = _lib.load()
    dev = _require_cuda("fused_moe_int4_ffn", A, w13_packed, w13_scale, w2_packed, w2_scale, topk_ids, topk_w, expert_map)
    if A.dtype not in _DT:
        raise TypeError(f"fused_moe_int4_ffn: A must be bf16 or fp32, got {A.dtype}")
    for name, t in (("w13_packed", w13_packed), ("w2_packed", w2_packed)):
        if t.dtype != torch.int32 or t.dim() != 3:
            raise TypeError(f"fused_moe_int4_ffn: {name} must be int32 [E, rows, K//8]")
    A, w13_packed, w2_packed = A.contiguous(), w13_packed.contiguous(), w2_packed.contiguous()
    M, hidden = A.shape
    E, two_inter, kp = w13_packed.shape
    inter = two_inter // 2
    group_size = int(group_size)
    if kp * 8 != hidden or two_inter % 2 or tuple(w2_packed.shape) != (E, hidden, inter // 8):
        raise ValueError("fused_moe_int4_ffn: w13_packed must be [E, 2*inter, hidden//8] and w2_packed [E, hidden, inter//8]")
    w13_scale = (w13_scale if w13_scale.dtype == torch.bfloat16 else w13_scale.to(torch.bfloat16)).contiguous()
    w2_scale = (w2_scale if w2_scale.dtype == torch.bfloat16 else w2_scale.to(torch.bfloat16)).contiguous()
    if tuple(w13_scale.shape) != (E, 2 * inter, hidden // group_size) or tuple(w2_scale.shape) != (E, hidden, inter // group_size):
        raise ValueError("fused_moe_int4_ffn: scale shapes must be [E, 2*inter, hidden//group] and [E, hidden, inter//group]")
    ids, tw, emap = _routing_args("fused_moe_int4_ffn", topk_ids, topk_w, expert_map, dev, M)
    top_k = ids.shape[1]
    limit = 0.0 if swiglu_limit is None else float(swiglu_limit)
    pcode = {"auto": _lib.PATH_AUTO, "simt": _lib.PATH_SIMT, "tc": _lib.PATH_TC}[path]
    if path != "simt":
        _check_int4_scales(w13_scale)
        _check_int4_scales(w2_scale)
    with _on(dev):
        out = torch.empty((M, hidden), dtype=A.dtype, device=dev)
        ws_bytes = _bytes("xkb_fused_moe_int4_ffn_workspace_bytes", M, hidden, inter, E, top_k, _DT[A.dtype])
        ws = _caller_workspace(workspace if isinstance(workspace, torch.Tensor) else None, False, ws_bytes, dev, ws_bytes)
        _lib.check(
            lib.xkb_fused_moe_int4_ffn(
                _ptr(A), _DT[A.dtype], _ptr(w13_packed), _ptr(w13_scale), _ptr(w2_packed), _ptr(w2_scale), _ptr(ids),
                _ptr(tw), _ptr(emap), 0 if emap is None else emap.numel(), _ptr(out), M, hidden, inter, E, top_k,
                group_size, limit, pcode, _ptr(ws), ws.numel(), _stream(dev)),
            "xkb_fused_moe_int4_ffn")
    return out


# ---------------------------------------------------------------------------
# expert-parallel building blocks
# ---------------------------------------------------------------------------
def moe_int4_w4a16_rows(A, packed, scale, topk_ids, topk_w=None, group_size=32, *, path="auto"):
    """Grouped INT4 expert GEMM without the top-k combine: ``[M*top_k, N]`` fp32 rows, row
    ``m*top_k + j`` = ``A[m] @ W[topk_ids[m,j]]^T`` (times ``topk_w[m,j]`` if given)."""
    lib = _lib.load()
    dev = _require_cuda("moe_int4_w4a16_rows", A, packed, scale, topk_ids, topk_w)
    if A.dtype not in _DT:
        raise TypeError(f"moe_int4_w4a16_rows: A must be bf16 or fp32, got {A.dtype}")
    A, packed = A.contiguous(), packed.contiguous()
    scale = scale.to(torch.bfloat16).contiguous()
    M, K = A.shape
    E, N, _ = packed.shape
    ids = topk_ids.to(torch.int32).contiguous()
    top_k = ids.shape[1]
    tw = None if topk_w is None else topk_w.to(torch.float32).contiguous()
    pcode = {"auto": _lib.PATH_AUTO, "simt": _lib.PATH_SIMT, "tc": _lib.PATH_TC}[path]
    if path != "simt":
        _check_int4_scales(scale)
    with _on(dev):
        rows = torch.empty((M * top_k, N), dtype=torch.float32, device=dev)
        if M == 0:
            return rows
        ws_bytes = _bytes("xkb_fused_moe_int4_w4a16_workspace_bytes", M, N, K, E, top_k, _DT[A.dtype])
        ws = get_workspace(dev, ws_bytes)
        _lib.check(
            lib.xkb_moe_int4_w4a16_rows(_ptr(A), _DT[A.dtype], _ptr(packed), _ptr(scale), _ptr(ids),
                                        _ptr(tw), _ptr(rows), M, N, K, E, top_k, int(group_size),
                                        0 if tw is None else 1, pcode, _ptr(ws), ws.numel(), _stream(dev)),
            "xkb_moe_int4_w4a16_rows")
    return rows


def moe_int4_w4a16_partial(A, packed, scale, routing, group_size=32, *, out=None, path="auto", workspace_tag=0):
    """Expert side of the all-to-all mode in one C call: ``A [R, K]`` received rows, ``routing
    [R, 2*top_k]`` int32 (local expert ids, -1 = elsewhere, then the routing weights' bit patterns)
    -> ``[R, N]`` fp32, per row the weighted sum over its local experts in ascending slot order (a
    row without a local expert comes out as zeros).  Two calls that overlap on different streams must
    use different ``workspace_tag`` values (see :func:`get_workspace`)."""
    lib = _lib.load()
    dev = _require_cuda("moe_int4_w4a16_partial", A, packed, scale, routing, out)
    if A.dtype not in _DT:
        raise TypeError(f"moe_int4_w4a16_partial: A must be bf16 or fp32, got {A.dtype}")
    if routing.dtype != torch.int32 or routing.dim() != 2 or routing.shape[1] % 2:
        raise TypeError("moe_int4_w4a16_partial: routing must be int32 [R, 2*top_k]")
    A, packed, routing = A.contiguous(), packed.contiguous(), routing.contiguous()
    scale = scale if scale.dtype == torch.bfloat16 else scale.to(torch.bfloat16)
    scale = scale.contiguous()
    R, K = A.shape
    E, N, _ = packed.shape
    top_k = routing.shape[1] // 2
    if routing.shape[0] != R:
        raise ValueError("moe_int4_w4a16_partial: one routing row per received row")
    pcode = {"auto": _lib.PATH_AUTO, "simt": _lib.PATH_SIMT, "tc": _lib.PATH_TC}[path]
    if path != "simt":
        _check_int4_scales(scale)
    with _on(dev):
        if out is None:
            out = torch.empty((R, N), dtype=torch.float32, device=dev)
        if out.dtype != torch.float32 or tuple(out.shape) != (R, N) or not out.is_contiguous():
            raise ValueError("moe_int4_w4a16_partial: out must be a contiguous fp32 [R, N] tensor")
        if R == 0:
            return out
        ws_bytes = _bytes("xkb_moe_int4_w4a16_partial_workspace_bytes", R, N, K, E, top_k, _DT[A.dtype])
        ws = get_workspace(dev, ws_bytes, tag=int(workspace_tag))
        _lib.check(
            lib.xkb_moe_int4_w4a16_partial(_ptr(A), _DT[A.dtype], _ptr(packed), _ptr(scale), _ptr(routing), _ptr(out),
                                           R, N, K, E, top_k, int(group_size), pcode, _ptr(ws), ws.numel(),
                                           _stream(dev)),
            "xkb_moe_int4_w4a16_partial")
    return out


def moe_gather_sum_reduce(rows, row_index, w, out_dtype=torch.bfloat16):
    """``out[m] = sum_k w[m,k] * rows[row_index[m,k]]`` in fp32, ascending k (index < 0 skips)."""
    lib = _lib.load()
    dev = _require_cuda("moe_gather_sum_reduce", rows, row_index, w)
    if rows.dtype != torch.float32:
        raise TypeError("moe_gather_sum_reduce: rows must be fp32")
    rows = rows.contiguous()
    idx = row_index.to(torch.int32).contiguous()
    M, top_k = idx.shape
    H = rows.shape[1]
    w = None if w is None else w.to(torch.float32).contiguous()
    with _on(dev):
        out = torch.empty((M, H), dtype=out_dtype, device=dev)
        _lib.check(
            lib.xkb_moe_gather_sum_reduce(_ptr(rows), _ptr(idx), _ptr(w), _ptr(out), _DT[out_dtype], M, top_k,
                                          H, _stream(dev)),
            "xkb_moe_gather_sum_reduce")
    return out


def gather_rows(src, index, count=None, out=None):
    """``out[p] = src[index[p]]`` for ``p < count[0]`` (``count`` a device int32 tensor; all of
    ``index`` if None).  ``out`` (``[>= len(index), row]``) may be a preallocated buffer; rows at and
    beyond the count are left untouched."""
    lib = _lib.load()
    dev = _require_cuda("gather_rows", src, index, count, out)
    src = src.contiguous()
    idx = index if index.dtype == torch.int32 else index.to(torch.int32)
    idx = idx.contiguous()
    row_bytes = src.shape[1] * src.element_size()
    n = idx.numel()
    with _on(dev):
        if out is None:
            out = torch.empty((n, src.shape[1]), dtype=src.dtype, device=dev)
        if out.dtype != src.dtype or out.shape[1] != src.shape[1] or out.shape[0] < n or not out.is_contiguous():
            raise ValueError("gather_rows: out must be a contiguous [>= len(index), row] tensor of src's dtype")
        _lib.check(lib.xkb_gather_rows(_ptr(src), src.shape[0], row_bytes, _ptr(idx), _ptr(count), n, _ptr(out),
                                       _stream(dev)), "xkb_gather_rows")
    return out


_PLACEMENT = {"contiguous": 0, "round_robin": 1, "snake": 2}


def ep_plan(topk_ids, topk_w, experts_per_rank, world, placement="contiguous", chunks=1, table=None):
    """Device-side dispatch plan of the all-to-all expert-parallel mode (``xkb_ep_plan``): no host
    read.  Returns ``(pair_token, pair_dest, routing, pair_of, counts, info)`` with the per-pair
    arrays sized ``M * top_k`` (the first ``info[0]`` entries are the pairs); see
    ``xkernels_b200/ep.py:plan_dispatch`` for the meaning of each.  ``table`` (``[E, 2]`` int32 on the
    device: destination rank and expert index there, per global expert) overrides ``placement``."""
    lib = _lib.load()
    dev = _require_cuda("ep_plan", topk_ids, topk_w)
    if placement not in _PLACEMENT:
        raise ValueError(f"unknown expert placement {placement!r}")
    ids = topk_ids.to(torch.int32).contiguous()
    w = topk_w.to(torch.float32).contiguous()
    M, top_k = ids.shape
    numel = M * top_k
    if table is not None:
        if table.dtype != torch.int32 or tuple(table.shape) != (int(experts_per_rank) * int(world), 2) or not table.is_cuda:
            raise ValueError("ep_plan: table must be a CUDA int32 tensor of shape [experts_per_rank * world, 2]")
        table = table.contiguous()
    with _on(dev):
        pair_token = torch.empty((numel,), dtype=torch.int32, device=dev)
        pair_dest = torch.empty((numel,), dtype=torch.int32, device=dev)
        routing = torch.empty((numel, 2 * top_k), dtype=torch.int32, device=dev)
        pair_of = torch.empty((M, world), dtype=torch.int32, device=dev)
        counts = torch.empty((chunks, world), dtype=torch.int32, device=dev)
        info = torch.empty((2,), dtype=torch.int32, device=dev)
        ws_bytes = _bytes("xkb_ep_plan_workspace_bytes", M, top_k, world, chunks)
        ws = get_workspace(dev, ws_bytes, tag=1)     # not the fused ops' buffer: that one starts with their status words
        _lib.check(
            lib.xkb_ep_plan(_ptr(ids), _ptr(w), M, top_k, int(experts_per_rank), int(world),
                            _PLACEMENT[placement], _ptr(table), int(chunks), _ptr(pair_token), _ptr(pair_dest),
                            _ptr(routing), _ptr(pair_of), _ptr(counts), _ptr(info), _ptr(ws), ws.numel(),
                            _stream(dev)),
            "xkb_ep_plan")
    return pair_token, pair_dest, routing, pair_of, counts, info
