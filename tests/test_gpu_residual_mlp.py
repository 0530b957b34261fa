"""The operators around the MLP block as a model uses them (examples/residual_mlp.py)."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")


def _example():
    sys.path.insert(0, EXAMPLES)
    try:
        import residual_mlp
    finally:
        sys.path.remove(EXAMPLES)
    return residual_mlp


def test_training_lowers_the_loss():
    losses = _example().train(width=128, hidden=512, depth=3, tokens=256, steps=40)
    assert losses[-1] < 0.5 * losses[0]


def test_gradients_of_the_stack():
    """Two blocks with odd sizes against the same model in fp32.  Bar: a bf16 rounding (2^-8) at each of the some ten
    results that follow one another from a weight to the loss and back, added up: 4e-2 of the 2-norm."""
    E = _example()
    torch.manual_seed(1)
    model = E.ResidualMLP(72, 200, 2)
    with torch.no_grad():
        for v in model.vectors():
            v.add_(0.2 * torch.randn_like(v))
    from bitsparse_amd.bitsparse import TensorBuffer
    x = torch.randn(100, 72, device="cuda").bfloat16().requires_grad_()
    g = torch.randn(100, 72, device="cuda").bfloat16()
    params = [x, *model.matrices(), *model.vectors()]
    got = torch.autograd.grad(model(x, TensorBuffer(4 * 100 * 200, device="cuda")), params, g)

    def norm(v, w):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w
    f = {id(p): p.detach().float().requires_grad_() for p in params}
    s = lambda p: f[id(p)]  # noqa: E731
    v = s(x)
    h = norm(v, s(model.pre[0]))
    for i in range(2):
        y = torch.relu(h @ s(model.up[i]).T).square() @ s(model.down[i]).T
        v = s(model.scale[i]) * v + s(model.gate[i]) * norm(y, s(model.post[i]))
        h = norm(v, s(model.pre[i + 1]))
    want = torch.autograd.grad(h, [s(p) for p in params], g.float())
    for a, b in zip(got, want):
        assert (a.float() - b).norm() < 4e-2 * b.norm(), (a.shape, ((a.float() - b).norm() / b.norm()).item())
