"""What stands between two MLP blocks of a residual stream: the norm before a
block, the norm after it with its gate, and the scaled residual.

``block_norm``: h = norm(x), a block's input.
``block_join``: from one block's output y to the next block's input, in one
pass over the rows (csrc/rownorm_fwd.hip; the gradients in one more,
csrc/rownorm_bwd.hip):

    p  = post(y)                   (y itself without ``post``), dropped out of with ``drop``
    x' = scale * x + gate * p      rounded to x's dtype
    h  = pre(x')                   of x' as stored, in y's dtype

A norm is c(v) / sqrt(mean(c(v)^2) + eps) * weight + bias over the last
dimension, with c(v) = v (``kind="rms"``) or v - mean(v) (``"layer"``).

A step of a residual model, each block's output joined and the next block's
input normalised by the same kernel::

    h = block_norm(x, norms[0])
    for i, (W1, W2) in enumerate(blocks):
        y = FFNRelu2.apply(h, W1, W2, sparse_data=buf)
        x, h = block_join(x, y, gate=gates[i], pre=norms[i + 1])
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from ._lib import native
from .dropout import Dropout, drop_parts

_KINDS = {"rms": 1, "layer": 2}


class RowNorm(NamedTuple):
    """A norm over the last dimension D.  weight, bias: [D] or None (1 and 0),
    bfloat16 or float32 each by itself."""
    weight: Tensor | None = None
    bias: Tensor | None = None
    kind: str = "rms"
    eps: float = 1e-6


_ABSENT = (None, None, 0, 0.0)


def _parts(norm: RowNorm | None, what: str) -> tuple:
    if norm is None:
        return _ABSENT
    weight, bias, kind, eps = norm
    if kind not in _KINDS:
        raise ValueError(f"{what}.kind must be 'rms' or 'layer', got {kind!r}")
    if not eps >= 0:
        raise ValueError(f"{what}.eps must not be negative, got {eps}")
    return weight, bias, _KINDS[kind], eps


def block_norm(x: Tensor, norm: RowNorm, *, dtype: torch.dtype | None = None) -> Tensor:
    """norm(x) over the last dimension, in ``dtype`` (x's by default; bfloat16
    of a float32 x for a block that takes it).

    x: [..., D], bfloat16 or float32, 0 < D <= 32768, rows of any stride.
    Differentiable once in x and the norm's vectors, in reverse mode; a tangent
    (forward mode) is refused."""
    weight, bias, kind, eps = _parts(norm, "norm")
    if kind == 0:
        raise TypeError("block_norm needs a RowNorm")
    dtype = x.dtype if dtype is None else dtype
    if dtype != torch.bfloat16 and dtype != torch.float32:
        raise TypeError(f"dtype must be bfloat16 or float32, got {dtype}")
    return native().join(x, None, None, None, None, None, weight, bias, 0, kind, 0.0, eps, 1.0, dtype)[0]


def block_join(x: Tensor, y: Tensor, *, post: RowNorm | None = None, gate: Tensor | None = None,
               scale: Tensor | float | None = None,
               pre: RowNorm | None = None, drop: Dropout | None = None) -> Tensor | tuple[Tensor, Tensor]:
    """x' = scale * x + gate * post(y), and with ``pre`` also h = pre(x').

    x: the residual stream [..., D]; y: the block's output, of the same shape.
    Both bfloat16, both float32, or a float32 x with a bfloat16 y.
    gate: None (1), one number (shape () or (1,)), a value a channel [D], a
    token [..., 1] or an element [..., D].
    scale: None (1), a Python number, or a tensor of one value or one a
    channel [D].
    drop: dropout of post(y), in front of the gate, with the mask that ``dropout`` has for [..., D] (fewer than 2^32 rows); none is stored.
    Returns x' (x's dtype), with ``pre`` the pair (x', h) (h in y's dtype).
    Differentiable once in every tensor, in reverse mode (a tangent is refused); the gradients are sums in 32 bits in
    a fixed order, each rounded once to its tensor's dtype."""
    w_post, b_post, kind_post, eps_post = _parts(post, "post")
    w_pre, b_pre, kind_pre, eps_pre = _parts(pre, "pre")
    if y is None:
        raise TypeError("block_join needs a block's output y; block_norm normalises x alone")
    value = 1.0
    if scale is not None and not isinstance(scale, Tensor):
        value, scale = float(scale), None
    args = (x, y, w_post, b_post, gate, scale, w_pre, b_pre, kind_post, kind_pre, eps_post, eps_pre, value, y.dtype)
    out = native().join(*args) if drop is None else native().join_drop(*args, *drop_parts(drop))
    return out[0] if pre is None else (out[0], out[1])
