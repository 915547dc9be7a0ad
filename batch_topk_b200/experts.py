"""Choosing experts for tokens and moving rows to them and back (tensor-level; ``torch_api``
re-exports it).

    weights, experts = route(logits, k, score="sigmoid", bias=bias, groups=8, topk_groups=4)
    plan = expert_order(experts, num_experts)        # the assignments sorted by expert
    rows = dispatch(x, plan)                         # [tokens * k, width], expert by expert
    ...                                              # the experts' products, rows
                                                     # plan.offsets[e]:plan.offsets[e + 1] for e
    y = combine(rows, plan, weights)                 # [tokens, width]

``route``, ``dispatch`` and ``combine`` have gradients.  Semantics, ties and empty slots are those
of the ``bt_`` entry points in include/batch_topk_b200.h.  No reference counterpart: the reference
ends with the top k (include/batch_topk.cuh:10-19).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import (MAX_ASSIGNMENTS, MAX_EXPERTS, MAX_EXPERTS_PER_TOKEN, SCORE_SIGMOID, SCORE_SOFTMAX,
               _lib)
from .sampling import ELEM, launch, raw_stream

SCORES = {"softmax": SCORE_SOFTMAX, "sigmoid": SCORE_SIGMOID}


class ExpertOrder(NamedTuple):
    """The assignments of [tokens, k] experts, sorted by expert (all int32).

    offsets [experts + 1]: expert e's assignments are order[offsets[e]:offsets[e + 1]];
    order [tokens * k]: which assignment (token * k + slot) stands at a place, -1 past the last;
    position [tokens, k]: the place of an assignment, -1 where its expert is none."""

    offsets: torch.Tensor
    order: torch.Tensor
    position: torch.Tensor


_workspaces: dict = {}


def _workspace(device, nbytes):
    """Scratch of the device's current stream, grown as needed: calls on one stream run in order,
    so they may share it; calls on different streams never do."""
    key = (device.index, raw_stream(device.index))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = _workspaces[key] = torch.empty(max(nbytes, 1 << 18), dtype=torch.uint8, device=device)
    return ws


def _first_order(grad):
    if grad.requires_grad:
        raise RuntimeError("route, dispatch and combine have first-order gradients only")


def _row_major(x):
    """x, or a copy whose rows are adjacent values (any row stride is fine)."""
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


def _check_rows(name, x):
    if x.dtype not in ELEM or x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{name} must be a 2-D float16, bfloat16 or float32 CUDA tensor")


def _route_forward(logits, k, score, bias, groups, topk_groups, renormalize, scale):
    tokens, experts = logits.shape
    dev = logits.device
    weights = torch.empty((tokens, k), dtype=torch.float32, device=dev)
    chosen = torch.empty((tokens, k), dtype=torch.int32, device=dev)
    if tokens:
        launch("route", _lib.load().bt_route, dev, logits.data_ptr(), ELEM[logits.dtype], tokens,
               experts, logits.stride(0), k, score, None if bias is None else bias.data_ptr(),
               groups, topk_groups, int(renormalize), scale, weights.data_ptr(),
               chosen.data_ptr())
    return weights, chosen


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, score, bias, groups, topk_groups, renormalize, scale):
        weights, chosen = _route_forward(logits, k, score, bias, groups, topk_groups, renormalize,
                                         scale)
        ctx.save_for_backward(logits, chosen)
        ctx.args = (k, score, renormalize, scale)
        ctx.mark_non_differentiable(chosen)
        ctx.set_materialize_grads(False)
        return weights, chosen

    @staticmethod
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * 8
        _first_order(grad)
        logits, chosen = ctx.saved_tensors
        k, score, renormalize, scale = ctx.args
        tokens, experts = logits.shape
        dev = logits.device
        out = torch.empty((tokens, experts), dtype=logits.dtype, device=dev)
        if tokens:
            grad = grad.float().contiguous()
            launch("route backward", _lib.load().bt_route_backward, dev, logits.data_ptr(),
                   ELEM[logits.dtype], tokens, experts, logits.stride(0), k, score,
                   int(renormalize), scale, chosen.data_ptr(), grad.data_ptr(), out.data_ptr())
        return out, None, None, None, None, None, None, None


def route(logits: torch.Tensor, k: int, *, score: str = "softmax",
          bias: torch.Tensor | None = None, groups: int = 1, topk_groups: int = 1,
          renormalize: bool = True, scale: float = 1.0):
    """(weights float32 [tokens, k], experts int32 [tokens, k]) of router logits
    [tokens, experts] (float16, bfloat16 or float32 on CUDA; rows may be strided).

    score: "softmax" or "sigmoid".  bias (float32 [experts]) is added to the scores for the choice
    alone.  groups > 1: only the topk_groups best of that many equal runs of experts stay in the
    choice.  renormalize: the chosen scores are divided by their sum.  scale multiplies the
    weights.  Slots for which no open expert is left hold expert -1 and weight 0.

    weights are differentiable in the logits.  Runs on the current stream of logits' device."""
    _check_rows("logits", logits)
    experts = logits.shape[1]
    if score not in SCORES:
        raise ValueError(f"score must be one of {sorted(SCORES)}, got {score!r}")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported, got {experts}")
    if not 1 <= groups <= 32 or experts % groups or not 1 <= topk_groups <= groups:
        raise ValueError(f"groups={groups}, topk_groups={topk_groups}: groups (at most 32) must "
                         f"divide {experts} experts, topk_groups must lie in [1, groups]")
    if not 1 <= k <= min(MAX_EXPERTS_PER_TOKEN, experts // groups * topk_groups):
        raise ValueError(f"k={k}: 1 to min({MAX_EXPERTS_PER_TOKEN}, experts that stay) are "
                         "supported")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (experts,)
                             or bias.device != logits.device):
        raise ValueError(f"bias must be a float32 tensor [{experts}] on {logits.device}")
    logits = _row_major(logits)
    bias = bias.detach().contiguous() if bias is not None else None
    args = (k, SCORES[score], bias, groups, topk_groups, renormalize, scale)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, *args)
    return _route_forward(logits, *args)


def expert_order(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The assignments of experts int32 [tokens, k] (CUDA) sorted by expert, equal experts in
    input order.  A number outside [0, num_experts), such as the -1 of an empty slot, is left out.
    Runs on the current stream of experts' device."""
    if experts.dtype != torch.int32 or experts.dim() != 2 or not experts.is_cuda:
        raise ValueError("experts must be a 2-D int32 CUDA tensor")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported, got {num_experts}")
    n = experts.numel()
    if n > MAX_ASSIGNMENTS:
        raise ValueError(f"at most {MAX_ASSIGNMENTS} assignments are supported, got {n}")
    dev = experts.device
    experts = experts.contiguous()
    if n == 0:
        return ExpertOrder(torch.zeros(num_experts + 1, dtype=torch.int32, device=dev),
                           torch.empty(0, dtype=torch.int32, device=dev),
                           torch.empty_like(experts))
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    order = torch.empty(n, dtype=torch.int32, device=dev)
    position = torch.empty_like(experts)
    lib = _lib.load()
    ws = _workspace(dev, lib.bt_expert_order_workspace_size(n, num_experts))
    launch("expert_order", lib.bt_expert_order, dev, experts.data_ptr(), n, num_experts,
           offsets.data_ptr(), order.data_ptr(), position.data_ptr(), ws.data_ptr(), ws.numel())
    return ExpertOrder(offsets, order, position)


def _check_plan(plan, device, tokens=None, rows=None):
    offsets, order, position = plan
    for name, t, dim in (("offsets", offsets, 1), ("order", order, 1), ("position", position, 2)):
        if t.dtype != torch.int32 or t.dim() != dim or t.device != device or not t.is_contiguous():
            raise ValueError(f"plan.{name} must be a contiguous {dim}-D int32 tensor on {device}")
    n, k = position.shape
    if order.numel() != n * k or offsets.numel() < 2:
        raise ValueError("plan.order must hold one place for each entry of plan.position")
    if not 1 <= k <= MAX_EXPERTS_PER_TOKEN or n * k > MAX_ASSIGNMENTS:
        raise ValueError(f"1 to {MAX_EXPERTS_PER_TOKEN} experts a token and at most "
                         f"{MAX_ASSIGNMENTS} assignments are supported, got {n} x {k}")
    if tokens is not None and tokens != n:
        raise ValueError(f"the plan is for {n} tokens, x has {tokens}")
    if rows is not None and rows != n * k:
        raise ValueError(f"the plan is for {n * k} rows, got {rows}")


def _dispatch(x, order, k):
    tokens, width = x.shape
    dev = x.device
    rows = torch.empty((tokens * k, width), dtype=x.dtype, device=dev)
    if rows.numel():
        launch("dispatch", _lib.load().bt_dispatch, dev, x.data_ptr(), ELEM[x.dtype], tokens, k,
               width, x.stride(0), order.data_ptr(), rows.data_ptr())
    return rows


def _combine(rows, position, weights):
    tokens, k = position.shape
    width = rows.shape[1]
    dev = rows.device
    y = torch.empty((tokens, width), dtype=rows.dtype, device=dev)
    if y.numel():
        launch("combine", _lib.load().bt_combine, dev, rows.data_ptr(), ELEM[rows.dtype], tokens, k,
               width, position.data_ptr(), None if weights is None else weights.data_ptr(),
               y.data_ptr())
    return y


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, position):
        ctx.save_for_backward(position)
        return _dispatch(x, order, position.shape[1])

    @staticmethod
    def backward(ctx, grad):
        _first_order(grad)
        position, = ctx.saved_tensors
        return _combine(grad.contiguous(), position, None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, offsets, position):
        ctx.save_for_backward(rows, weights, offsets, position)
        return _combine(rows, position, weights)

    @staticmethod
    def backward(ctx, grad):
        _first_order(grad)
        rows, weights, offsets, position = ctx.saved_tensors
        tokens, k = position.shape
        dev = rows.device
        d_rows = torch.empty_like(rows) if ctx.needs_input_grad[0] else None
        d_weights = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        if rows.numel():
            grad = _row_major(grad)
            live = offsets.data_ptr() + 4 * (offsets.numel() - 1)
            launch("combine backward", _lib.load().bt_combine_backward, dev, rows.data_ptr(),
                   grad.data_ptr(), ELEM[rows.dtype], tokens, k, rows.shape[1], grad.stride(0),
                   position.data_ptr(), live, weights.data_ptr(),
                   None if d_rows is None else d_rows.data_ptr(),
                   None if d_weights is None else d_weights.data_ptr())
        elif d_weights is not None:
            d_weights.zero_()
        return d_rows, d_weights, None, None


def dispatch(x: torch.Tensor, plan: ExpertOrder) -> torch.Tensor:
    """The rows of x [tokens, width] (float16, bfloat16 or float32 on CUDA; rows may be strided)
    in the experts' order: [tokens * k, width], zeros past the last assignment.  Differentiable in
    x.  Runs on the current stream of x's device."""
    _check_rows("x", x)
    _check_plan(plan, x.device, tokens=x.shape[0])
    x = _row_major(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, plan.order, plan.position)
    return _dispatch(x, plan.order, plan.position.shape[1])


def combine(rows: torch.Tensor, plan: ExpertOrder, weights: torch.Tensor) -> torch.Tensor:
    """The weighted sum of each token's rows: [tokens, width] in the rows' type, summed in 32 bits,
    from rows [tokens * k, width] in the experts' order and weights float32 [tokens, k].  An
    assignment without an expert adds nothing, and its weight's gradient is 0.  Differentiable in
    rows and weights.  Runs on the current stream of rows' device."""
    _check_rows("rows", rows)
    _check_plan(plan, rows.device, rows=rows.shape[0])
    if (weights.dtype != torch.float32 or weights.shape != plan.position.shape
            or weights.device != rows.device):
        raise ValueError("weights must be a float32 tensor of plan.position's shape on the rows' "
                         "device")
    rows = rows.contiguous()
    weights = weights.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad):
        return _Combine.apply(rows, weights, plan.offsets, plan.position)
    return _combine(rows, plan.position, weights)
