"""The operators around a block have no forward-mode derivative: a tensor with a tangent is refused, since a result
without one would read as a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad

from bitsparse_amd.muon import muon_update_, orthogonalize
from bitsparse_amd.residual import RowNorm, block_join, block_norm

BF = torch.bfloat16


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def _calls(x, y, v, m):
    """name, operand -> the call with it as one of its operands"""
    n, t = RowNorm(v), v.clone()
    yield "x of the norm", x, lambda d: block_norm(d, n)
    yield "weight", t, lambda d: block_norm(x, RowNorm(d))
    yield "bias", t, lambda d: block_norm(x, RowNorm(v, d))
    yield "x", x, lambda d: block_join(d, y, pre=n)
    yield "y", y, lambda d: block_join(x, d)
    yield "post", t, lambda d: block_join(x, y, post=RowNorm(d))
    yield "gate", t, lambda d: block_join(x, y, gate=d)
    yield "gate by row", x[:, :1], lambda d: block_join(x, y, gate=d)
    yield "scale", t, lambda d: block_join(x, y, scale=d)
    yield "G", m, lambda d: orthogonalize(d)
    yield "a gradient", m, lambda d: muon_update_([m.clone()], [d], [m.clone()], lr=0.1)


@pytest.mark.parametrize("requires_grad", [False, True])
def test_refused_before_the_device(requires_grad):
    """On any device (here the CPU's, whose tensors are otherwise refused for that)."""
    x = torch.ones(4, 64, dtype=BF)
    with forward_ad.dual_level():
        d = _dual(x.clone().requires_grad_(requires_grad))
        for call in (lambda: block_norm(d, RowNorm()), lambda: block_join(d, x), lambda: orthogonalize(d)):
            with pytest.raises(NotImplementedError):
                call()


@pytest.mark.gpu
def test_refused_in_every_operand():
    x, y = (torch.randn(4, 64, device="cuda").to(BF) for _ in range(2))
    v, m = torch.rand(64, device="cuda"), torch.randn(8, 12, device="cuda")
    for name, t, call in _calls(x, y, v, m):
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                call(_dual(t))
                pytest.fail(name)
        call(t)                     # without a tangent it runs


@pytest.mark.gpu
def test_tangent_of_a_gradient():
    x = torch.randn(4, 64, device="cuda").to(BF).requires_grad_()
    h = block_norm(x, RowNorm())
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(h, x, _dual(torch.ones_like(h)))


@pytest.mark.gpu
def test_forward_mode_switched_off():
    """Inside a level with forward mode off, a tensor that has a tangent is an ordinary one."""
    x = torch.randn(4, 64, device="cuda")
    want = block_norm(x, RowNorm())
    with forward_ad.dual_level():
        d = _dual(x)
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(block_norm(d, RowNorm()), want)
