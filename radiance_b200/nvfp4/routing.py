"""Token routing around the grouped expert linears (``grouped.py``): picks, balance loss, and the
moves of token rows to the experts' rows and back.

radiance's ``MoEFeedForward`` (src/radiance/model/ffn.py:156-436) routes with softmax, topk and index
ops.  Here ``route`` makes one pass over the logits: the picks and their weights, the experts' counts,
the balance loss, and the rows of the expert-sorted layout that ``FP4GroupedLinear`` multiplies
(groups padded to 128 rows).  ``token_dispatch`` and ``token_combine`` move the rows.  Counts and
offsets stay on the device; nothing synchronises with the host.  All results, gradients included,
repeat bit for bit.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from . import _trace
from .epilogue import _call, _dtype_of, _first_order, _like, _rows, _size, _tracked
from .quantize import _require_cuda

MAX_EXPERTS = 256  # the grouped GEMM's group limit
MAX_TOP_K = 32


class Routing(NamedTuple):
    """One batch's routing (``route``).  ``rows[t, j]`` is the expert-sorted row of token t's pick j."""

    weights: torch.Tensor  # (tokens, k) fp32, differentiable; 0 where there is no pick
    experts: torch.Tensor  # (tokens, k) int32; -1 where there is no pick
    counts: torch.Tensor  # (experts,) int64: pairs of each expert
    balance_loss: torch.Tensor  # 0-d fp32, differentiable
    offsets: torch.Tensor  # (experts + 1,) int64: first row of each expert's group, for FP4GroupedLinear
    rows: torch.Tensor  # (tokens, k) int32; -1 where there is no pick
    num_rows: int  # rows of the expert-sorted tensors: enough for any routing of this size
    # The counts that the row moves go by, in a tensor of their own: `counts` may be changed in place (an all-reduce
    # over a data-parallel job's ranks) at any time.  A plan with other counts or offsets sets it, or None for `counts`.
    plan_counts: torch.Tensor | None = None


def routed_rows(tokens: int, k: int, experts: int) -> int:
    """Rows that any routing of these sizes fits in, every expert's group padded to a multiple of 128."""
    pairs = tokens * k
    return (pairs + 127 * min(experts, pairs)) // 128 * 128


def _route(logits, k, expert_bias, valid, renormalize):
    what = "nvfp4.route"
    code = _dtype_of(logits, what)
    logits, ld = _rows(logits)
    tokens, experts = logits.shape
    dev = logits.device
    weights = torch.empty(tokens, k, dtype=torch.float32, device=dev)
    # Tensors of their own: what a caller does to one in place (an all-reduce of the counts) leaves the others'
    # versions alone.  The backward reads `share`, which no caller sees, instead of the counts, and the row moves
    # read `plan_counts`.
    picks = torch.empty(tokens, k, dtype=torch.int32, device=dev)
    rows = torch.empty(tokens, k, dtype=torch.int32, device=dev)
    counts = torch.empty(experts, dtype=torch.int64, device=dev)
    plan_counts = torch.empty(experts, dtype=torch.int64, device=dev)
    offsets = torch.empty(experts + 1, dtype=torch.int64, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    share = torch.empty(experts, dtype=torch.float32, device=dev)
    lib = _lib.load()
    need = _size(dev, lib.rb_nvfp4_route_workspace, tokens, experts, k)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    tok = _trace.begin("route", logits.numel() * logits.element_size() + 12 * tokens * k)
    _call(what, dev, lib.rb_nvfp4_route_plan, logits.data_ptr(), code, tokens, experts, ld, k,
          None if expert_bias is None else expert_bias.data_ptr(), None if valid is None else valid.data_ptr(),
          int(renormalize), weights.data_ptr(), picks.data_ptr(), rows.data_ptr(), counts.data_ptr(),
          plan_counts.data_ptr(), offsets.data_ptr(), loss.data_ptr(), share.data_ptr(), ws.data_ptr(), need)
    _trace.end(tok)
    return weights, loss, picks, counts, offsets, rows, plan_counts, share


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, expert_bias, valid, renormalize):
        ctx.set_materialize_grads(False)
        *out, share = _route(logits, k, expert_bias, valid, renormalize)
        weights, _, picks = out[:3]
        ctx.mark_non_differentiable(*out[2:])
        ctx.save_for_backward(logits, weights, picks, share)
        ctx.renormalize, ctx.curved = renormalize, True
        return tuple(out)

    @staticmethod
    @_first_order
    def backward(ctx, grad_w, grad_loss, *_):
        if grad_w is None and grad_loss is None:
            return None, None, None, None, None
        what = "nvfp4.route backward"
        logits, weights, picks, share = ctx.saved_tensors
        tokens, experts = logits.shape
        grad = torch.empty(tokens, experts, dtype=logits.dtype, device=logits.device)
        x, ld = _rows(logits)
        if grad_w is not None:
            grad_w = grad_w.contiguous()
        tok = _trace.begin("route", 2 * x.numel() * x.element_size() + 12 * picks.numel())
        _call(what, x.device, _lib.load().rb_nvfp4_route_backward, x.data_ptr(), _dtype_of(x, what), tokens, experts,
              ld, picks.shape[1], int(ctx.renormalize), weights.data_ptr(), picks.data_ptr(), share.data_ptr(),
              None if grad_w is None else grad_w.data_ptr(), None if grad_loss is None else grad_loss.data_ptr(),
              grad.data_ptr(), experts)
        _trace.end(tok)
        return grad, None, None, None, None


def route(logits: torch.Tensor, k: int, *, expert_bias: torch.Tensor | None = None,
          valid: torch.Tensor | None = None, renormalize: bool = True) -> Routing:
    """Top-``k`` routing of ``(tokens, experts)`` router logits (bf16 or fp32), one pass.

    A token's picks are the k experts of largest ``logit + expert_bias`` (fp32; ties go to the lower
    expert; ``expert_bias`` steers the selection only).  Its weights are the softmax of its logits at the
    picks, divided by their sum with ``renormalize``.  ``balance_loss`` is
    ``E * sum_e f_e P_e``: ``f_e`` the expert's share of all pairs, ``P_e`` its mean probability over the
    routed tokens (1 when both are uniform).  Gradients flow from ``weights`` and ``balance_loss`` to
    the logits, with the selection and the counts held constant.

    An expert with score -inf is never picked; a token left with fewer than k experts has picks of -1
    with weight 0.  A token left with none, or with ``valid`` (bool, one per token) false, is not
    routed: its logits are ignored, whatever they hold, and their gradient is 0.
    """
    what = "nvfp4.route"
    _require_cuda(logits, what)
    _dtype_of(logits, what)
    if logits.dim() != 2:
        raise ValueError(f"{what}: logits must be (tokens, experts), got shape {tuple(logits.shape)}")
    tokens, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= k <= min(experts, MAX_TOP_K):
        raise ValueError(f"{what}: needs 1 <= experts <= {MAX_EXPERTS} and 1 <= k <= min(experts, {MAX_TOP_K}), got "
                         f"experts={experts} k={k}")
    if expert_bias is not None:
        _like("expert_bias", expert_bias, (experts,), expert_bias.dtype, logits.device, what)
        expert_bias = expert_bias.detach().to(torch.float32).contiguous()
    if valid is not None:
        _like("valid", valid, (tokens,), torch.bool, logits.device, what)
        valid = valid.contiguous()
    if _tracked(logits):
        out = _RouteFn.apply(logits, k, expert_bias, valid, renormalize)
    else:
        out = _route(logits, k, expert_bias, valid, renormalize)[:-1]
    weights, loss, picks, counts, offsets, rows, plan_counts = out
    return Routing(weights, picks, counts, loss, offsets, rows, routed_rows(tokens, k, experts), plan_counts)


# ------------------------------------------------------------------------------------------------
# Rows
# ------------------------------------------------------------------------------------------------


def _plan(r: Routing, device: torch.device, what: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(rows, counts, offsets) of a routing, checked."""
    rows, counts, offsets = r.rows, r.counts if r.plan_counts is None else r.plan_counts, r.offsets
    if rows.dtype != torch.int32 or counts.dtype != torch.int64 or offsets.dtype != torch.int64 or rows.dim() != 2 \
            or counts.dim() != 1 or offsets.shape != (counts.shape[0] + 1,):
        raise ValueError(f"{what}: the routing needs int32 rows (tokens, k) and int64 counts (E,) and offsets (E + 1,)")
    if rows.device != device or counts.device != device or offsets.device != device:
        raise ValueError(f"{what}: the routing is on {rows.device}, the rows on {device}")
    if rows.shape[1] < 1 or r.num_rows < 0:
        raise ValueError(f"{what}: the routing needs at least one pick per token and num_rows >= 0")
    return rows.contiguous(), counts.contiguous(), offsets.contiguous()


def _dispatch(x, rows, counts, offsets, num_rows):
    what = "nvfp4.token_dispatch"
    x, ld = _rows(x)
    tokens, d = x.shape
    out = torch.empty(num_rows, d, dtype=x.dtype, device=x.device)
    tok = _trace.begin("rows", (x.numel() + out.numel()) * x.element_size())
    _call(what, x.device, _lib.load().rb_nvfp4_token_dispatch, x.data_ptr(), _dtype_of(x, what), tokens, d, ld,
          rows.data_ptr(), rows.shape[1], counts.data_ptr(), offsets.data_ptr(), counts.numel(), out.data_ptr(),
          num_rows, d)
    _trace.end(tok)
    return out


def _combine(y, rows, weights, residual):
    what = "nvfp4.token_combine"
    y, ld = _rows(y)
    num_rows, d = y.shape
    tokens, k = rows.shape
    ldr = d
    if residual is not None:
        residual, ldr = _rows(residual)
    out = torch.empty(tokens, d, dtype=y.dtype, device=y.device)
    tok = _trace.begin("rows", (tokens * (k + 1 + (residual is not None))) * d * y.element_size())
    _call(what, y.device, _lib.load().rb_nvfp4_token_combine, y.data_ptr(), _dtype_of(y, what), num_rows, d, ld,
          rows.data_ptr(), k, None if weights is None else weights.data_ptr(),
          None if residual is None else residual.data_ptr(), ldr, out.data_ptr(), tokens, d)
    _trace.end(tok)
    return out


def _combine_backward(grad_y, y, rows, weights, counts, offsets):
    what = "nvfp4.token_combine backward"
    y, ldy = _rows(y)
    grad_y, ldg = _rows(grad_y)
    num_rows, d = y.shape
    tokens, k = rows.shape
    grad_rows = torch.empty(num_rows, d, dtype=y.dtype, device=y.device)
    grad_w = torch.empty(tokens, k, dtype=torch.float32, device=y.device)
    tok = _trace.begin("rows", (tokens * (k + 1) + num_rows) * d * y.element_size())
    _call(what, y.device, _lib.load().rb_nvfp4_token_combine_backward, grad_y.data_ptr(), ldg, y.data_ptr(), ldy,
          _dtype_of(y, what), tokens, d, rows.data_ptr(), k, weights.data_ptr(), counts.data_ptr(),
          offsets.data_ptr(), counts.numel(), grad_rows.data_ptr(), num_rows, d, grad_w.data_ptr())
    _trace.end(tok)
    return grad_rows, grad_w


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rows, counts, offsets, num_rows):
        ctx.save_for_backward(rows)
        return _dispatch(x, rows, counts, offsets, num_rows)

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        (rows,) = ctx.saved_tensors
        return _combine(grad, rows, None, None), None, None, None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, rows, counts, offsets):
        ctx.save_for_backward(y, weights, rows, counts, offsets)
        ctx.curved = ctx.needs_input_grad[0] and ctx.needs_input_grad[1]  # each one's gradient depends on the other
        return _combine(y, rows, weights, residual)

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        y, weights, rows, counts, offsets = ctx.saved_tensors
        gy = gw = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            gy, gw = _combine_backward(grad, y, rows, weights, counts, offsets)
        return gy, gw, (grad if ctx.needs_input_grad[2] else None), None, None, None


def token_dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Token rows ``(tokens, d)`` in the expert-sorted layout ``(routing.num_rows, d)``: every pick's row
    holds its token, every other row is zero (``FP4GroupedLinear``'s input, with ``routing.offsets``).
    Differentiable in ``x``: the gradient is the sum over the token's picks.  bf16 or fp32, any d."""
    what = "nvfp4.token_dispatch"
    _require_cuda(x, what)
    _dtype_of(x, what)
    rows, counts, offsets = _plan(routing, x.device, what)
    if x.dim() != 2 or x.shape[0] != rows.shape[0] or x.shape[1] < 1:
        raise ValueError(f"{what}: rows of shape ({rows.shape[0]}, d) expected, got {tuple(x.shape)}")
    if _tracked(x):
        return _DispatchFn.apply(x, rows, counts, offsets, routing.num_rows)
    return _dispatch(x, rows, counts, offsets, routing.num_rows)


def token_combine(y: torch.Tensor, routing: Routing, *, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + sum_j weights[t, j] * y[rows[t, j]]``: expert rows ``(num_rows, d)`` back to tokens
    ``(tokens, d)``, summed in fp32 in the order of the picks and rounded once.  A token without picks gets
    its residual (or 0); rows of ``y`` that hold no pick are never read.  Differentiable in ``y`` (the
    gradient of those rows is 0), ``routing.weights`` and ``residual``."""
    what = "nvfp4.token_combine"
    _require_cuda(y, what)
    _dtype_of(y, what)
    rows, counts, offsets = _plan(routing, y.device, what)
    tokens, k = rows.shape
    if y.dim() != 2 or y.shape[0] != routing.num_rows or y.shape[1] < 1:
        raise ValueError(f"{what}: expert rows of shape ({routing.num_rows}, d) expected, got {tuple(y.shape)}")
    weights = routing.weights
    _like("routing.weights", weights, (tokens, k), torch.float32, y.device, what)
    weights = weights.contiguous()
    if residual is not None:
        _like("residual", residual, (tokens, y.shape[1]), y.dtype, y.device, what)
    if _tracked(y, weights, residual):
        return _CombineFn.apply(y, weights, residual, rows, counts, offsets)
    return _combine(y, rows, weights, residual)
