"""What an optimiser step leaves in the momentum."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(*s, seed=0):
    return torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("mu", [0.0, 0.5, 0.9, 0.95, 0.999, 0.9999])
@pytest.mark.parametrize("shape", [(40, 70), (129, 33)])
def test_momentum_in_32_bits(mu, shape):
    """M' = mu M + (1 - mu) G of the mu that was given.  Bar: mu and 1 - mu rounded, two products and a sum, each to
    2^-24: four roundings of each term at most."""
    from bitsparse_amd.muon import muon_update_
    G, W = _randn(*shape, seed=1), _randn(*shape, seed=2)
    for M in (torch.zeros(shape, device="cuda"), _randn(*shape, seed=3)):
        old, fresh = mu * M.double(), (1 - mu) * G.double()
        muon_update_([W], [G], [M], lr=0.1, momentum=mu)
        assert ((M.double() - (old + fresh)).abs() <= 4 * 2.0 ** -24 * (old.abs() + fresh.abs())).all()


@pytest.mark.parametrize("eps", [-1e-3, -1e30, float("nan")])
def test_eps(eps):
    """An X_0 past a norm of 1 would leave the operands' range unseen: refused, with nothing touched."""
    from bitsparse_amd.muon import muon_update_, orthogonalize
    G = _randn(20, 30)
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(G, eps=eps)
    W, M = G.clone(), G.clone()
    with pytest.raises(ValueError, match="eps"):
        muon_update_([W], [G], [M], lr=0.1, eps=eps)
    assert torch.equal(W, G) and torch.equal(M, G)
    assert orthogonalize(G, eps=0.0).isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,C", [(200, 300), (300, 200), (1, 5000)])
def test_norm_past_fp32(dtype, R, C):
    """Elements near fp32's largest, whose norm is past it: a power of two off, the same bits (eps counts in neither)."""
    from bitsparse_amd.muon import orthogonalize
    G = (_randn(R, C).clamp(-3, 3) * 2.0 ** 126 / 3).to(dtype)
    assert torch.equal(orthogonalize(G), orthogonalize(G * 2.0 ** -60)) and orthogonalize(G).any()
