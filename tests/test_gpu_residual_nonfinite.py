"""Infinities and NaNs in the step between two blocks: a result that the formulas give as a finite number or as an
infinity is that, whatever stands beside it.  Bar of the finite ones: one rounding to the result's type (half a unit,
2^-8 in bf16 and 2^-24 in fp32) and 2^-19 of the terms' magnitudes for the 32-bit arithmetic before it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def _mod():
    from bitsparse_amd import residual
    return residual


def _same(got, want, mag, name):
    """Finite where `want` is, and close; the same infinities and NaNs elsewhere."""
    got = got.double()
    fin = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), name
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), name
    half = 2.0 ** -8 if name.endswith("bf16") else 2.0 ** -24
    bad = (got - want).abs()[fin] > half * want.abs()[fin] * (1 + 2.0 ** -6) + 2.0 ** -19 * mag[fin]
    assert not bad.any(), (name, int(bad.sum()))


def _randn(*s, seed=0):
    return torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(seed + sum(s)), device="cuda")


SHAPES = {"one": lambda T, D: (1,), "channel": lambda T, D: (D,), "row": lambda T, D: (T, 1), "element": lambda T, D: (T, D)}


@pytest.mark.parametrize("T,D", [(5, 64), (7, 2001), (3, 5000)])
@pytest.mark.parametrize("gate", [None, "one", "channel", "row", "element"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_of_a_block_output_that_overflowed(T, D, gate, dtype):
    """Without a norm after the block dy = gate dx', whatever y is."""
    x, y, g = (_randn(T, D, seed=i).to(dtype) for i in range(3))
    y[0, 3], y[1, 5], y[2, 7] = math.inf, -math.inf, math.nan
    gv = None if gate is None else (0.5 + 0.3 * _randn(*SHAPES[gate](T, D), seed=3))
    y.requires_grad_()
    x1 = _mod().block_join(x, y, gate=gv)
    dy, = torch.autograd.grad(x1, y, g)
    want = g.double() * (1.0 if gv is None else gv.double())
    _same(dy, want, want.abs(), "dy " + ("bf16" if dtype == BF else "fp32"))


@pytest.mark.parametrize("T,D", [(5, 64), (7, 2001), (3, 9000)])
@pytest.mark.parametrize("gate", ["one", "channel", "row", "element"])
@pytest.mark.parametrize("post,bias", [(None, False), ("rms", False), ("layer", False), ("rms", True), ("layer", True)])
@pytest.mark.parametrize("big", [math.inf, -math.inf, math.nan])
def test_gates_past_the_range(T, D, gate, post, bias, big):
    """x' = scale x + gate p: an infinite gate gives infinities of p's sign, not NaN, also where p is the sum of two
    terms of different signs."""
    R = _mod()
    x, y = _randn(T, D), _randn(T, D, seed=1)
    gv = 0.5 + 0.3 * _randn(*SHAPES[gate](T, D), seed=3)
    gv.view(-1)[::3] = big
    w, b = 1 + 0.2 * _randn(D, seed=4), 0.5 * _randn(D, seed=5)
    x1 = R.block_join(x, y, post=R.RowNorm(w, b if bias else None, post, EPS) if post else None, gate=gv, scale=0.75)
    p, mag = y.double(), y.double().abs()
    if post:
        c = p - p.mean(-1, keepdim=True) if post == "layer" else p
        r = 1 / ((c * c).mean(-1, keepdim=True) + EPS).sqrt()
        b = b.double() if bias else torch.zeros((), dtype=torch.float64, device="cuda")
        mag = (mag + mag.mean(-1, keepdim=True)) * r * w.double().abs() + b.abs()
        p = c * r * w.double() + b
    want = 0.75 * x.double() + gv.double() * p
    _same(x1, want, 0.75 * x.double().abs() + (gv.double() * mag).abs().nan_to_num(posinf=0.0), "x1 fp32")


@pytest.mark.parametrize("post", ["rms", "layer"])
def test_gradient_of_one_gate_with_an_infinite_gradient(post):
    """dgate = sum G p is infinite where one G is; the bias that is not there adds nothing to it."""
    R = _mod()
    x, y, g = (_randn(9, 300, seed=i) for i in range(3))
    g[4, 100] = math.inf
    gv = torch.full((1,), 0.5, device="cuda").requires_grad_()
    x1 = R.block_join(x, y, post=R.RowNorm(None, None, post, EPS), gate=gv)
    d, = torch.autograd.grad(x1, gv, g)
    c = y - y.mean(-1, keepdim=True) if post == "layer" else y
    assert d.item() == math.copysign(math.inf, c[4, 100].item())
