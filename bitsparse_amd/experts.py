"""MLP blocks as experts: the routing of tokens, the products of each expert's
rows with its weights, and the weighted sum back to tokens.

    w, experts = route(x @ Wr.T, top_k)               # [T, k] each
    plan = plan_experts(experts, n_experts)           # rows by expert
    out = ExpertsRelu2.apply(x, W1, W2, w, plan, sparse_data=buf)

or, step by step,

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
from torch.autograd import Function

from ._lib import native
from .bitsparse import BitsparseTensor, TensorBuffer
from .config import RELU2_SCALE
from .src.functions import relu2_and_compress, relu2_fused_ok, relu_and_compress
from .src.hip_operators import relu2_square_amax_
from .src.sparse_matmul import decoded

_SCORES = {"softmax": 0, "sigmoid": 1}


class ExpertPlan(NamedTuple):
    """The routed (token, choice) pairs in the order of their experts, int32:
    rows offsets[e] up to offsets[e + 1] belong to expert e, order[row] is the
    pair token * top_k + choice, place[token, choice] its row, -1 where it has
    none.  offsets[e0:e1 + 1] with W[e0:e1] is the plan of a part of the
    experts: rows before the first offset and from the last on are of none."""
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
    its rows need it; W: [E, d_out, d_in]; both bfloat16.  Rows of no
    expert, behind the last one's or before the first one's, are 0, and the
    gradients of x (as x is given) and W take nothing from them.  Sums in 32 bits, each result rounded once.  Differentiable once in x and W."""
    return native().expert_linear(x, W, *plan, gather)


def expert_combine(y: Tensor, weights: Tensor, plan: ExpertPlan) -> Tensor:
    """out[token] = sum over its choices of weights[token, choice] * y[its
    row], [..., d_out]; choices without a row of an expert add nothing.

    y: bfloat16 [rows, d_out]; weights: float32 [..., top_k].  Sums in 32 bits
    in the order of the choices.  Differentiable once in y and weights."""
    return native().expert_combine(y, weights, *plan)


# ------------------------------------------------------------
# blocks of experts whose activation is saved compressed
# ------------------------------------------------------------
class ExpertsRelu:
    """FFNRelu as experts: the weighted sum over a token's experts of
    relu(x @ W1[e].T) @ W2[e].T."""

    @staticmethod
    def apply(x: Tensor, W1: Tensor, W2: Tensor, weights: Tensor, plan: ExpertPlan, *,
              sparse_data: TensorBuffer | None = None, pack_sbit: bool = False) -> Tensor:
        """x [..., d_in], W1 [E, d_ff, d_in], W2 [E, d_out, d_ff], all bfloat16; weights float32 [..., top_k] and the plan as
        ``route`` and ``plan_experts`` give them -> [..., d_out].

        The activation of all rows [tokens * top_k, d_ff] is saved compressed, as the dense blocks save theirs (``sparse_data``,
        ``pack_sbit``); the second product's result is not saved at all.  Without a gradient to come nothing is, and the
        activation is part of the first product.  Differentiable once in x, W1, W2 and weights."""
        return _experts(x, W1, W2, weights, plan, sparse_data, pack_sbit, False)


class ExpertsRelu2:
    """FFNRelu2 as experts: the weighted sum over a token's experts of
    k * relu(x @ W1[e].T)^2 @ W2[e].T.  Arguments as ``ExpertsRelu``'s."""

    @staticmethod
    def apply(x: Tensor, W1: Tensor, W2: Tensor, weights: Tensor, plan: ExpertPlan, *,
              sparse_data: TensorBuffer | None = None, pack_sbit: bool = False) -> Tensor:
        return _experts(x, W1, W2, weights, plan, sparse_data, pack_sbit, True)


def _experts(x, W1, W2, weights, plan, sparse_data, pack_sbit, square) -> Tensor:
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, W1, W2, weights)):
        return _ExpertsBlock.apply(x, W1, W2, weights, *plan, sparse_data, pack_sbit, square)
    h = native().expert_product(x, W1, *plan, True, 2 if square else 1, float(RELU2_SCALE))
    return native().expert_combine(native().expert_product(h, W2, *plan, False, 0, 0.0), weights, *plan)


class _ExpertsBlock(Function):
    @staticmethod
    def forward(ctx, x, W1, W2, weights, offsets, order, place, sparse_data, pack_sbit, square):
        plan = (offsets, order, place)
        h, ctx.h_sparse = _activate(native().expert_product(x, W1, *plan, True, 0, 0.0), sparse_data, pack_sbit, square)
        ctx.square = square
        ctx.save_for_backward(x, W1, W2, weights, *plan)
        return native().expert_combine(native().expert_product(h, W2, *plan, False, 0, 0.0), weights, *plan)

    @staticmethod
    @torch.compiler.disable
    def backward(ctx, grad_output: Tensor):
        if torch.is_grad_enabled():
            raise NotImplementedError("bitsparse_amd: a block of experts has no second derivative (create_graph)")
        if ctx.h_sparse is None:
            raise RuntimeError("a block of experts goes backward once: its compressed activation is freed with it")
        h = ctx.h_sparse
        r = decoded(h, False) if h.shape[0] else grad_output.new_empty(h.shape)
        del h
        ctx.h_sparse = None
        grads = native().experts_backward(grad_output, *ctx.saved_tensors, r, ctx.square, float(RELU2_SCALE), ctx.needs_input_grad[:4])
        return *grads, None, None, None, None, None, None


def _activate(z: Tensor, sparse_data: TensorBuffer | None, pack_sbit: bool, square: bool) -> tuple[Tensor, BitsparseTensor]:
    """(the activation of z, which it overwrites; relu(z) compressed)"""
    if square and relu2_fused_ok(z, sparse_data, pack_sbit, RELU2_SCALE):
        return z, relu2_and_compress(z, sparse_data, RELU2_SCALE)
    h, h_sparse = relu_and_compress(z, sparse_data, pack_sbit)
    if square:
        relu2_square_amax_(h, RELU2_SCALE)
    return h, h_sparse
