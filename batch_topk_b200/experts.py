"""Choosing experts for tokens and moving rows to them and back (tensor-level; ``torch_api``
re-exports it).

    weights, experts = route(logits, k, score="sigmoid", bias=bias, groups=8, topk_groups=4)
    plan = expert_order(experts, num_experts)        # the assignments sorted by expert
    rows = dispatch(x, plan)                         # [tokens * k, width], expert by expert
    ...                                              # the experts' products, rows
                                                     # plan.offsets[e]:plan.offsets[e + 1] for e
    y = combine(rows, plan, weights)                 # [tokens, width]

``route``, ``dispatch`` and ``combine`` have first-order gradients; forward-mode derivatives and
differentiating a gradient again raise a RuntimeError.  Semantics, ties and empty slots are those of
the ``bt_`` entry points in include/batch_topk_b200.h.  No reference counterpart: the reference
ends with the top k (include/batch_topk.cuh:10-19).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import tensors


class ExpertOrder(NamedTuple):
    """The assignments of [tokens, k] experts, sorted by expert (all int32).

    offsets [experts + 1]: expert e's assignments are order[offsets[e]:offsets[e + 1]];
    order [tokens * k]: which assignment (token * k + slot) stands at a place, -1 past the last;
    position [tokens, k]: the place of an assignment, -1 where its expert is none.

    order and position are each other's inverse, which the gradients of dispatch and combine rely
    on."""

    offsets: torch.Tensor
    order: torch.Tensor
    position: torch.Tensor


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
    return tensors().route(logits, k, score, bias, groups, topk_groups, renormalize, scale)


def expert_order(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The assignments of experts int32 [tokens, k] (CUDA) sorted by expert, equal experts in
    input order.  A number outside [0, num_experts), such as the -1 of an empty slot, is left out.
    Runs on the current stream of experts' device."""
    return ExpertOrder(*tensors().expert_order(experts, num_experts))


def dispatch(x: torch.Tensor, plan: ExpertOrder) -> torch.Tensor:
    """The rows of x [tokens, width] (float16, bfloat16 or float32 on CUDA; rows may be strided)
    in the experts' order: [tokens * k, width], zeros past the last assignment.  Differentiable in
    x.  Runs on the current stream of x's device."""
    return tensors().dispatch(x, plan)


def combine(rows: torch.Tensor, plan: ExpertOrder, weights: torch.Tensor) -> torch.Tensor:
    """The weighted sum of each token's rows: [tokens, width] in the rows' type, summed in 32 bits,
    from rows [tokens * k, width] in the experts' order and weights float32 [tokens, k].  An
    assignment without an expert adds nothing, and its weight's gradient is 0.  Differentiable in
    rows and weights.  Runs on the current stream of rows' device."""
    return tensors().combine(rows, plan, weights)
