"""Orthogonalised updates of weight matrices.

``orthogonalize(G)``: U V^T-like factor of G = U S V^T by Newton-Schulz
products on the matrix cores (csrc/newton.hip): X = G / (||G||_F + eps), then
``steps`` times X <- a X + (b A + c A^2) X with A = X X^T.  With the default
coefficients every singular value that is not tiny beside the others comes to
0.7 .. 1.2, not to 1 itself.

``muon_update_``: a whole optimiser step of a list of matrices -- momentum,
orthogonalisation, weight decay, step -- in place; matrices of one shape (and
their transposes) go through each product together.  ``Muon`` is the
optimiser around it.

Precision: products of fp16 operands (11 bits) summed in fp32, a choice for
speed where bf16 takes the result.  For gradients of full rank it is within
1-3e-3 (2-norm) of the exact iteration's, of which 1.7e-3 is the rounding to
bf16.  Where a gradient has directions of no gradient at all (fewer tokens t
than rows), the iteration raises the operands' rounding noise there, to about
0.16 / sqrt(t) of the result: for 768 x 3072 2.4e-3 at 768 tokens, 3.2e-3 at
576, 9e-3 at 192, 2e-2 at 64 and 0.15 at one (products of fp32 operands: 3e-6
to 2e-4).  ``precise`` holds every operand as two fp16 numbers and multiplies
three times: 2e-6, 1.4e-5 at 192 tokens and 1e-4 at one, before the result's own rounding,
at a third of the speed; updates of float32 weights do so unless told
otherwise, and it is the form for gradients of few tokens.
"""
from __future__ import annotations

from typing import Sequence

import torch
from torch import Tensor

from ._lib import native

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(G: Tensor, *, steps: int = 5, coefficients: tuple[float, float, float] = COEFFICIENTS,
                  eps: float = 1e-7, precise: bool = False) -> Tensor:
    """The orthogonalised matrices of G [..., R, C] (bfloat16 or float32, up to
    65536 rows and columns and fewer than 2^29 elements each), in bfloat16, contiguous.

    ``precise``: products of 22-bit operands (see above).  Coefficients that
    could take X, A, b A + c A^2 + a or b X + c A X past 15 raise ValueError.  No gradient flows
    through it (an optimiser's operator), and a tangent is refused."""
    a, b, c = coefficients
    with torch.no_grad():
        return native().orthogonalize(G, steps, a, b, c, eps, precise)


def muon_update_(params: Sequence[Tensor], grads: Sequence[Tensor], momenta: Sequence[Tensor], *, lr: float,
                 momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 adjust: str | float = "shape", steps: int = 5,
                 coefficients: tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7,
                 precise: bool | None = None) -> None:
    """For each matrix W [R, C] with its gradient G and momentum M, in place:

        M <- momentum M + (1 - momentum) G
        U  = (1 - momentum) G + momentum M  (nesterov)  or  M
        W <- (1 - lr weight_decay) W - lr s orthogonalize(U)

    s: sqrt(max(1, R / C)) (``adjust="shape"``), 0.2 sqrt(max(R, C))
    (``"rms"``: updates of the size that Adam's have) or the number given.
    precise: products of 22-bit operands, by default for float32 weights.
    Each of the three lists is bfloat16 or float32; W and M have contiguous
    rows, their own memory (shared with no other matrix of the lists; a G with its own W
    at most), and are updated on the current stream."""
    if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
        raise ValueError(f"lr and weight_decay must not be negative and momentum be in [0, 1), got lr={lr}, "
                         f"weight_decay={weight_decay}, momentum={momentum}")
    if isinstance(adjust, str):
        if adjust not in ("shape", "rms"):
            raise ValueError(f"adjust must be 'shape', 'rms' or a number, got {adjust!r}")
        by_rms, scale = adjust == "rms", -1.0
    else:
        by_rms, scale = False, float(adjust)
        if not scale >= 0:
            raise ValueError(f"adjust must not be negative, got {adjust}")
    a, b, c = coefficients
    with torch.no_grad():
        native().muon_update(list(params), list(grads), list(momenta), lr, momentum, nesterov, weight_decay, by_rms,
                             scale, steps, a, b, c, eps, precise)


class Muon(torch.optim.Optimizer):
    """``muon_update_`` as an optimiser of weight matrices (an MLP block's W1
    and W2); vectors and embeddings belong to another one.

        opt = Muon([W1, W2], lr=0.02)
        loss.backward(); opt.step(); opt.zero_grad()

    The momentum is kept in ``momentum_dtype`` (float32 by default)."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 adjust: str | float = "shape", steps: int = 5, coefficients: tuple[float, float, float] = COEFFICIENTS,
                 eps: float = 1e-7, momentum_dtype: torch.dtype = torch.float32, precise: bool | None = None):
        if momentum_dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"momentum_dtype must be float32 or bfloat16, got {momentum_dtype}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      adjust=adjust, steps=steps, coefficients=coefficients, eps=eps,
                                      momentum_dtype=momentum_dtype, precise=precise))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon updates matrices, got a parameter of shape {tuple(p.shape)}")

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (torch casts a parameter's state to the parameter's dtype: the momentum has its own)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, (p, dtype) in zip(ids, ((p, g["momentum_dtype"]) for g in self.param_groups for p in g["params"])):
            if "momentum" in state_dict["state"].get(i, {}):
                self.state[p]["momentum"] = state_dict["state"][i]["momentum"].detach().to(p.device, dtype, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            for p in params:
                if "momentum" not in self.state[p]:
                    self.state[p]["momentum"] = torch.zeros(p.shape, dtype=group["momentum_dtype"], device=p.device)
            muon_update_(params, [p.grad for p in params], [self.state[p]["momentum"] for p in params],
                         **{k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "adjust", "steps",
                                                  "coefficients", "eps", "precise")})
        return loss
