"""How many matrices go through the Newton-Schulz products together."""
import pytest
import torch

from bitsparse_amd import _lib

GIB = 1 << 30
COEF = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("rows,cols", [(4096, 16384), (16384, 4096), (2048, 5500), (768, 3072), (64, 64), (8192, 65535), (1, 65536)])
@pytest.mark.parametrize("precise", [0, 1])
def test_scratch_is_bounded(rows, cols, precise):
    """A list of any length takes 1 GiB and a little (the partial sums), or what one matrix takes."""
    need = _lib.load().bs_newton_schulz_workspace_bytes
    one = need(rows, cols, 1, precise)
    for count in (2, 3, 30, 64, 65, 72, 1000):
        assert one <= need(rows, cols, count, precise) <= max(one, GIB) + (320 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("B,R,C,precise", [(3, 4096, 16384, False), (3, 2048, 16000, True), (72, 768, 3072, False), (65, 100, 250, True)])
def test_groups(B, R, C, precise):
    """Each matrix of a list that goes in groups is what it is alone: two results, each within 2e-3 of the exact one (of
    which half a unit of bf16 makes 1.7e-3)."""
    from bitsparse_amd.muon import orthogonalize
    G = torch.randn(B, R, C, generator=torch.Generator(device="cuda").manual_seed(B), device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = orthogonalize(G, precise=precise)
    assert torch.cuda.max_memory_allocated() - before - 2 * G.numel() < GIB + (320 << 20)
    for i in {0, 1, B // 2, B - 2, B - 1}:
        alone = orthogonalize(G[i], precise=precise).float()
        assert (got[i].float() - alone).norm() < 4e-3 * alone.norm(), i
    assert torch.equal(got, orthogonalize(G, precise=precise))


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(32768, 32768), (16384, 65536), (8, 65537)])
def test_refused_before_memory_is_taken(R, C):
    """(a view that takes no memory itself)"""
    from bitsparse_amd.muon import muon_update_, orthogonalize
    G = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(R, C)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(ValueError, match="65536"):
        orthogonalize(G)
    with pytest.raises(ValueError):
        muon_update_([G], [G], [G], lr=0.1)
    assert torch.cuda.max_memory_allocated() == before


@pytest.mark.gpu
@pytest.mark.parametrize("adjust", ["shape", "rms", 0.3])
def test_transposes_go_together(adjust):
    """W1 [H, D] and W2 [D, H] of two blocks in one call of the products, whatever the scale of each one's step: the call's
    scratch is that of four matrices.  Each is stepped as orthogonalize says, both in half a unit of bf16 (2^-8 at most, and
    1.7e-3 of the 2-norm) and 1e-3 of the exact one."""
    import math

    from bitsparse_amd.muon import muon_update_, orthogonalize
    D, H = 256, 1024
    g = torch.Generator(device="cuda").manual_seed(3)
    shapes = [(H, D), (D, H), (H, D), (D, H)]
    G = [torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in shapes]
    W = [torch.zeros(s, device="cuda", dtype=torch.bfloat16) for s in shapes]
    M = [torch.zeros(s, device="cuda") for s in shapes]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    muon_update_(W, G, M, lr=0.5, momentum=0.0, adjust=adjust)
    assert torch.cuda.max_memory_allocated() - before >= _lib.load().bs_newton_schulz_workspace_bytes(D, H, 4, 0)
    for w, x, (r, c) in zip(W, G, shapes):
        s = {"shape": math.sqrt(max(1, r / c)), "rms": 0.2 * math.sqrt(max(r, c))}.get(adjust, adjust)
        want = -0.5 * s * orthogonalize(x).float()
        assert (w.float() - want).norm() < 5.4e-3 * want.norm()
