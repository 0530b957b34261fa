"""Matrices of an optimiser step that share memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(*s, seed=0):
    return torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _update(W, G, M):
    from bitsparse_amd.muon import muon_update_
    muon_update_(W, G, M, lr=0.1)


def test_refused():
    """What is written twice, or read after another matrix's write: refused before anything is touched."""
    buf, g, m = _randn(60, 40), _randn(20, 30, seed=1), _randn(20, 30, seed=2)
    own = lambda: torch.zeros(20, 30, device="cuda")  # noqa: E731
    a, b, shifted = buf[:20, :30], buf[20:40, :30], buf[10:30, 5:35]
    for W, G, M in (([a, a], [g, g], [m, own()]), ([a, shifted], [g, g], [m, own()]), ([a], [g], [shifted]), ([a, b], [g, g], [m, m]),
                    ([a], [m], [m]), ([a, b], [own(), m], [m, own()]), ([a, b], [g, a], [m, own()]), ([a, b], [shifted, g], [m, own()]),
                    ([buf[:, :30]], [buf[:, 3:33]], [buf[:, 8:38]])):
        before = [t.clone() for t in (buf, g, m)]
        with pytest.raises(ValueError, match="share memory"):
            _update(W, G, M)
        assert all(torch.equal(t, u) for t, u in zip((buf, g, m), before))


def test_apart():
    """Columns of one buffer between each other's, rows behind each other, gradients shared by several matrices or
    with their own parameter: as with memory of their own."""
    buf, g = _randn(40, 90), _randn(40, 30, seed=1)
    both = _randn(40, 30, seed=3)
    for W, G, M in (([buf[:, :30], buf[:, 30:60]], [g, g], [torch.zeros(40, 30, device="cuda"), buf[:, 60:]]),
                    ([buf[:20, :30], buf[20:, :30]], [g[:20], g[20:]], [buf[:20, 30:60], buf[20:, 30:60]]),
                    ([both], [both], [buf[:, :30]]), ([buf[:, :30]], [_randn(1, 30, seed=4).expand(40, 30)], [buf[:, 31:61]])):
        apart = [[t.clone() for t in ts] for ts in (W, G, M)]
        if W[0].data_ptr() == G[0].data_ptr():
            apart[1] = [t.clone() for t in apart[0]]
        _update(*apart)
        _update(W, G, M)
        assert all(torch.equal(t, u) for ts, us in zip((W, M), (apart[0], apart[2])) for t, u in zip(ts, us))


def test_inference_tensors():
    """Not updated outside inference mode, like any tensor made there: refused before the first matrix is touched."""
    with torch.inference_mode():
        made = torch.randn(20, 30, device="cuda")
    for k in range(2):
        W, G, M = (_randn(20, 30, seed=i) for i in range(3))
        V = W.clone()
        lists = ([W, made], [G, G], [M, V]) if k == 0 else ([W, V], [G, G], [M, made])
        before = [t.clone() for t in (W, M, V, made)]
        with pytest.raises(RuntimeError, match="inference"):
            _update(*lists)
        assert all(torch.equal(t, u) for t, u in zip((W, M, V, made), before))
    with torch.inference_mode():
        W, N = made.clone(), made.clone()
        _update([W], [G], [N])
        assert not torch.equal(W, made)
