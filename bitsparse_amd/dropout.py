"""Dropout whose mask is a function of a seed and an element's place, so that
none is stored: the backward pass forms the forward's again.

``dropout`` of any tensor; ``residual.block_join`` takes the same rule for a
block's output on its way into the residual stream.  Element (row, column) of
the rows [..., D] is kept where its 16 bits of Philox 4x32 (10 rounds; key
seed, counter (column / 8, row, offset)) are at least round(65536 p), and is
then scaled by 65536 / (65536 - round(65536 p)) (csrc/philox.h).

A training step's blocks each take their own offset::

    y = FFNRelu2.apply(h, W1, W2, sparse_data=buf)
    x, h = block_join(x, y, drop=Dropout(0.1, seed, step * n_blocks + i), pre=norms[i + 1])
"""
from __future__ import annotations

from typing import NamedTuple

from torch import Tensor

from ._lib import native


class Dropout(NamedTuple):
    """p: share of the elements that are dropped, taken to the nearest 1/65536.
    seed, offset: any numbers below 2^64; each pair has a mask of its own, and
    tensors that are to have independent masks take different ones.  seed may
    be an int64 tensor [seed, offset] on the values' device instead, which a
    captured graph reads at every replay; it must not change between a
    forward pass and its backward."""
    p: float
    seed: int | Tensor
    offset: int = 0


def drop_parts(drop: Dropout) -> tuple:
    """(bound, seed, offset, state) for the native calls"""
    if not isinstance(drop, Dropout):
        raise TypeError(f"drop must be a Dropout, got {type(drop).__name__}")
    if not 0.0 <= drop.p <= 1.0:
        raise ValueError(f"drop.p must be in 0..1, got {drop.p}")
    below = round(65536 * drop.p)
    if isinstance(drop.seed, Tensor):
        if drop.offset != 0:
            raise ValueError("drop.offset: a tensor drop.seed holds the offset too")
        return below, 0, 0, drop.seed
    for name, value in (("seed", drop.seed), ("offset", drop.offset)):
        if not 0 <= value < 2 ** 64:
            raise ValueError(f"drop.{name} must be in 0..2^64-1, got {value}")
    return below, drop.seed, drop.offset, None


def dropout(x: Tensor, drop: Dropout) -> Tensor:
    """x with elements dropped (0, whatever they were) and the others scaled.

    x: bfloat16 or float32 on the GPU, any shape and strides; its last
    dimension is a row, of which there are fewer than 2^32.  The result is
    contiguous.  Differentiable in x any number of times, in reverse mode."""
    return native().dropout(x, *drop_parts(drop))
