"""MLP blocks as experts: the routing of tokens, the products of each expert's
rows with its weights, and the weighted sum back to tokens.

    w, experts = route(x @ Wr.T, top_k)               # [T, k] each
    plan = plan_experts(experts, n_experts)           # rows by expert
    z = expert_linear(x, W1, plan, gather=True)       # [T k, d_ff], by expert
    y = expert_linear(act(z), W2, plan)               # [T k, d_out]
    out = expert_combine(y, w, plan)                  # [T, d_out]

The routing stays on the device: no step waits for how many rows an expert
gets (csrc/route.hip, csrc/experts_gemm.hip, csrc/experts_rows.hip).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from ._lib import native

_SCORES = {"softmax": 0, "sigmoid": 1}


class ExpertPlan(NamedTuple):
    """The routed (token, choice) pairs in the order of their experts, int32:
    rows offsets[e] up to offsets[e + 1] belong to expert e, order[row] is the
    pair token * top_k + choice, place[token, choice] its row, -1 where it has
    none."""
    offsets: Tensor
    order: Tensor
    place: Tensor


def route(logits: Tensor, top_k: int, *, score: str = "softmax", bias: Tensor | None = None, groups: int = 1,
          top_groups: int | None = None, group_best: int = 1, renormalize: bool = True,
          scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """The experts of each token and their weights, float32 and int32 [..., top_k], the largest first.

    logits: [..., E], bfloat16 or float32, E <= 1024, top_k <= 64; s is their
    softmax or sigmoid.  Experts are chosen by s + bias (bias: float32 [E], for
    balance; it has no part in the weights and no gradient), with ``groups``
    among the experts of the ``top_groups`` groups (all by default) whose
    ``group_best`` (1 or 2) best ones have the largest sum; of equal ones the
    lower index.  The choice is as between 64-bit values (between the logits
    themselves where the order is theirs).  weights = scale * s, divided by the sum over the
    token's choices with ``renormalize``.
    An expert whose logit (or whose biased score) is -inf is not chosen; a choice left without
    one is -1 with weight 0, which is how a padded token (all -inf) goes nowhere.  A NaN counts as +inf.
    Differentiable once in logits."""
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    top_groups = groups if top_groups is None else top_groups
    w, experts = native().route(logits, bias, top_k, _SCORES[score], groups, top_groups, group_best, renormalize, scale)
    return w, experts


def plan_experts(experts: Tensor, n_experts: int) -> ExpertPlan:
    """Where the pairs of ``experts`` (int32 [..., top_k]) go: sorted by
    expert, those of one expert in their own order.  Ids outside
    0..n_experts-1 (padding, another rank's experts) get no row."""
    return ExpertPlan(*native().plan_experts(experts, n_experts))


def expert_linear(x: Tensor, W: Tensor, plan: ExpertPlan, *, gather: bool = False) -> Tensor:
    """y[row] = x[row] @ W[expert of row].T, [rows, d_out], rows as in ``plan``.

    x: [rows, d_in], or with ``gather`` the tokens [..., d_in], each read where
    its rows need it; W: [E, d_out, d_in]; both bfloat16.  Rows behind the last
    expert's are 0, and the gradients of x (as x is given) and W take nothing
    from them.  Sums in 32 bits, each result rounded once.  Differentiable once in x and W."""
    return native().expert_linear(x, W, *plan, gather)


def expert_combine(y: Tensor, weights: Tensor, plan: ExpertPlan) -> Tensor:
    """out[token] = sum over its choices of weights[token, choice] * y[its
    row], [..., d_out]; choices without a row add nothing.

    y: bfloat16 [rows, d_out]; weights: float32 [..., top_k].  Sums in 32 bits
    in the order of the choices.  Differentiable once in y and weights."""
    return native().expert_combine(y, weights, *plan)
