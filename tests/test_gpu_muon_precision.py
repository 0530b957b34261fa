"""How far orthogonalised gradients may be off, where the bf16 result does not hide it and where gradients lack rank."""
import math

import pytest
import torch

from tests.test_gpu_muon import _err, _exact, _grads, _model22

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


# the products that take 22-bit operands: 256 x 256 and 128 x 128 tiles with their last round shared and without, 64 x 64
# and 32 x 32 tiles, a long K split over workgroups, the kernel of few rows, lists that go in groups with plans of their own
SHAPES = [(2, 2048, 5500), (1, 2304, 4700), (3, 1000, 3100), (2, 1024, 4100), (12, 768, 3072), (65, 768, 3072), (1, 300, 16000),
          (1, 64, 8200), (3, 200, 9000), (1, 16000, 190), (65, 200, 70), (5, 256, 256)]


@pytest.mark.parametrize("B,R,C", SHAPES)
def test_22_bits(B, R, C):
    """Into fp32 weights of 0, so that nothing is rounded to bf16.  Bar: twice the distance of a model with the same
    roundings, plus 2^-20 for sums in another order (operands without their low parts are 1e-3 off)."""
    from bitsparse_amd.muon import muon_update_
    G = _grads(B, R, C, 21)
    wide = G if R <= C else G.mT.contiguous()
    W, M = torch.zeros_like(G), torch.zeros_like(G)
    muon_update_(list(W), list(G), list(M), lr=1.0, momentum=0.0, adjust=1.0)
    got = -(W if R <= C else W.mT)
    for i in range(0, B, 8):
        want = _exact(wide[i:i + 8])
        model = _err(_model22(wide[i:i + 8]), want)
        err = _err(got[i:i + 8], want)
        assert err <= 2 * model + 2.0 ** -20, (i, err, model)


def _of_tokens(R, C, tokens, seed=0):
    """The gradient of a Linear's weight: outputs' gradients times a ReLU's outputs, summed over tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    dy = rn(R, tokens) * torch.exp(0.5 * rn(R, 1))
    return dy @ torch.relu(rn(tokens, C) + 0.3 * rn(1, C))


@pytest.mark.parametrize("R,C", [(768, 1536), (1000, 700), (256, 1024)])
@pytest.mark.parametrize("share", [1 / 64, 1 / 12, 1 / 4, 3 / 4, 2])
def test_fewer_tokens_than_rows(R, C, share):
    """Directions without a gradient: each step raises what rounding puts there by a = 3.44.  X_0 and its successors of
    norm min(3.44^k, sqrt(t)) are rounded to 2^-12.2 (the root mean square of 11 bits), raised by 3.44^(5 - k): root of the
    sum of squares under 940 2^-12.2 = 0.2 beside a result of norm sqrt(t).  2e-3 more: the full-rank error and bf16's."""
    from bitsparse_amd.muon import orthogonalize
    t = max(1, round(share * min(R, C)))
    G = _of_tokens(R, C, t)
    want = _exact((G if R <= C else G.T.contiguous())[None])[0]
    want = want if R <= C else want.T
    t = min(t, R, C)
    err = ((orthogonalize(G).double() - want).norm() / want.norm()).item()
    precise = ((orthogonalize(G, precise=True).double() - want).norm() / want.norm()).item()
    assert err <= 0.2 / math.sqrt(t) + 2e-3, err
    assert precise <= 0.2 * 2.0 ** -11 / math.sqrt(t) + 2e-3, precise
