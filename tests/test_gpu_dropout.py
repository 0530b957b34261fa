"""Dropout from the counter-based generator, alone and in the step between two blocks, against its definition.

Bars: a result is rounded once, 2^-8 (bf16) or 2^-24 (fp32) of its value at
most, the scale 65536 / (65536 - q) once more (2^-24); the step's as in
tests/test_gpu_residual.py, 2^-19 of the sum of its terms' magnitudes.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def kept(rows, cols, below, seed, offset):
    """Which elements stay: Philox 4x32, 10 rounds, on the host in 64-bit integers."""
    n = (cols + 7) // 8
    c = [np.broadcast_to(v, (len(rows), n)).astype(np.uint64) for v in
         (np.arange(n)[None], np.asarray(rows)[:, None], np.uint64(offset % 2 ** 32), np.uint64(offset >> 32))]
    k0, k1 = seed % 2 ** 32, seed >> 32
    low, w = np.uint64(2 ** 32 - 1), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> w) ^ c[1] ^ np.uint64(k0), b & low, (a >> w) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    u = np.stack([h for v in c for h in (v & np.uint64(65535), v >> np.uint64(16))], -1).reshape(len(rows), -1)[:, :cols]
    return u >= below


def test_generator_known_answer():
    """The published test vector of Philox 4x32-10: counter and key all ones bits (Random123's kat_vectors)."""
    c, k0, k1 = [2 ** 32 - 1] * 4, 2 ** 32 - 1, 2 ** 32 - 1
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k0, b % 2 ** 32, (a >> 32) ^ c[3] ^ k1, a % 2 ** 32]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    assert c == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def _close(got, want, mag=None):
    half = 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    tol = half * want.abs() * (1 + 2.0 ** -6) + (2.0 ** -23 * want.abs() if mag is None else 2.0 ** -19 * mag) + 1e-37
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3].tolist(), want[bad][:3].tolist())


SEEDS = [(0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (0x123456789abcdef0, 5 << 33)]


@pytest.mark.parametrize("T,D,p", [(1, 1, 0.5), (1, 4096, 0.1), (257, 100, 0.1), (33, 7, 0.9), (1000, 768, 0.2), (3, 8193, 0.5), (4096, 1, 0.25)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("seed,offset", SEEDS)
def test_dropout(T, D, p, dtype, seed, offset):
    from bitsparse_amd.dropout import Dropout, dropout
    x = torch.randn(T, D + 3, device="cuda").to(dtype)[:, :D].requires_grad_()
    drop = Dropout(p, seed, offset)
    out = dropout(x, drop)
    q = round(65536 * p)
    m = torch.from_numpy(kept(range(T), D, q, seed, offset)).cuda()
    want = m * x.detach().double() * (65536 / (65536 - q))
    _close(out.detach(), want)
    assert torch.equal(out == 0, ~m | (x == 0))
    g = torch.randn(T, D, device="cuda").to(dtype)
    dx, = torch.autograd.grad(out, x, g)
    _close(dx, m * g.double() * (65536 / (65536 - q)))


def test_dropout_ends_of_its_range():
    from bitsparse_amd.dropout import Dropout, dropout
    x = torch.randn(50, 60, device="cuda")
    assert torch.equal(dropout(x, Dropout(0.0, 3)), x)
    x[3], x[4] = torch.inf, torch.nan
    assert (dropout(x, Dropout(1.0, 3)) == 0).all()
    y = dropout(x, Dropout(0.5, 3))
    m = torch.from_numpy(kept(range(50), 60, 32768, 3, 0)).cuda()
    assert (y[3] == torch.where(m[3], torch.inf, 0.0)).all() and torch.equal(y[4].isnan(), m[4]) and (y[4][~m[4]] == 0).all()
    for shape in ((0, 5), (5, 0), (), (3,), (2, 3, 4)):
        t = torch.randn(shape, device="cuda")
        out = dropout(t, Dropout(0.5, 3))
        assert out.shape == t.shape


def test_dropout_share_and_scale():
    """The share that stays is p's within five standard deviations, and the mean is kept."""
    from bitsparse_amd.dropout import Dropout, dropout
    n = 1 << 22
    for p in (0.1, 0.5, 0.9):
        y = dropout(torch.ones(1024, n // 1024, device="cuda"), Dropout(p, 11, 12))
        sd = (p * (1 - p) / n) ** 0.5
        assert abs((y == 0).double().mean().item() - p) < 5 * sd + 2.0 ** -17
        assert abs(y.double().mean().item() - 1) < 5 * sd / (1 - p) + 1e-6


def test_dropout_state_on_the_device():
    from bitsparse_amd.dropout import Dropout, dropout
    x = torch.randn(40, 130, device="cuda").requires_grad_()
    for seed, offset in ((5, 6), (2 ** 63 - 1, 2 ** 40 + 1)):
        state = torch.tensor([seed, offset], device="cuda")
        a, b = dropout(x, Dropout(0.3, state)), dropout(x, Dropout(0.3, seed, offset))
        assert torch.equal(a, b)
        ga, = torch.autograd.grad(a, x, torch.ones_like(a), retain_graph=True)
        assert torch.equal(ga, torch.autograd.grad(b, x, torch.ones_like(b))[0])
        state += 1                      # a backward after this would have another mask
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(a, x, torch.ones_like(a))


def test_dropout_second_derivative():
    from bitsparse_amd.dropout import Dropout, dropout
    x = torch.randn(20, 24, device="cuda").requires_grad_()
    drop = Dropout(0.4, 9)
    g, = torch.autograd.grad((dropout(x, drop) ** 2).sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), x)
    m = torch.from_numpy(kept(range(20), 24, round(65536 * 0.4), 9, 0)).cuda()
    s = 65536 / (65536 - round(65536 * 0.4))
    assert torch.allclose(h.double(), m.double() * (2 * s * s), rtol=2.0 ** -21)


# ---------------------------------------------------------------------------
# in the step between two blocks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,D", [(1, 8), (5, 100), (64, 768), (37, 2501), (9, 4096), (7, 5000), (3, 9000), (2, 20001)])
@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (F32, F32)])
@pytest.mark.parametrize("post,gate", [(None, None), ("rms", "channel"), ("layer", "row"), (None, "element"), ("rms", "one"), ("layer", "channel")])
def test_join_with_dropout(T, D, xt, yt, post, gate):
    """The step with its dropout is the step on what dropout alone makes of p: the formulas in 64 bits with the same mask."""
    from bitsparse_amd.dropout import Dropout
    from bitsparse_amd.residual import RowNorm, block_join
    g = torch.Generator(device="cuda").manual_seed(T + D)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    drop = Dropout(0.3, 77, 2 ** 35 + D)
    q = round(65536 * 0.3)
    t = {"x": rn(T, D).to(xt), "y": rn(T, D).to(yt), "w_pre": (1 + 0.2 * rn(D)).to(xt)}
    if post:
        t["w_post"], t["b_post"] = (1 + 0.2 * rn(D)).to(xt), (0.1 * rn(D)).to(xt)
    if gate:
        t["gate"] = (0.5 + 0.3 * rn(*{"one": (1,), "channel": (D,), "row": (T, 1), "element": (T, D)}[gate])).to(yt if gate == "element" else xt)
    for v in t.values():
        v.requires_grad_()
    x1, h = block_join(t["x"], t["y"], post=RowNorm(t["w_post"], t["b_post"], post, 1e-5) if post else None, gate=t.get("gate"), scale=0.9,
                       pre=RowNorm(t["w_pre"], None, "rms", 1e-5), drop=drop)
    gx, gh = rn(T, D).to(xt), rn(T, D).to(yt)
    grads = dict(zip(t, torch.autograd.grad((x1, h), list(t.values()), (gx, gh))))

    v = {k: a.detach().double().requires_grad_() for k, a in t.items()}
    m = torch.from_numpy(kept(range(T), D, q, drop.seed, drop.offset)).cuda().double() * (65536 / (65536 - q))
    yn = v["y"]
    if post:
        c = yn - yn.mean(-1, keepdim=True) if post == "layer" else yn
        yn = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    p = yn * v["w_post"] + v["b_post"] if post else yn
    gate64 = v["gate"] if gate else 1.0
    ref = 0.9 * v["x"] + gate64 * m * p
    # how large the terms are that the results are formed of
    size = 0.9 * v["x"].abs().detach() + ((gate64.abs() if gate else 1.0) * m * p.abs()).detach()
    _close(x1.detach(), ref.detach(), size + (size.mean(-1, keepdim=True) if post else 0.0))
    stored = ref + (x1.detach().double() - ref.detach())
    hr = stored * torch.rsqrt((stored * stored).mean(-1, keepdim=True) + 1e-5) * v["w_pre"]
    _close(h.detach(), hr.detach(), hr.detach().abs())
    want = dict(zip(v, torch.autograd.grad((stored, hr), list(v.values()), (gx.double(), gh.double()))))
    for k in t:
        # (the sums over rows and columns that a gradient has part in: bounded by their root mean square and extent)
        w = want[k]
        n = T if w.numel() in (D, 1) else 1
        n = n * (D if w.numel() in (1, T) else 1)
        rms = w.square().mean().sqrt()
        tol = (2.0 ** -8 if grads[k].dtype == BF else 2.0 ** -24) * w.abs() * 1.02 + 2.0 ** -17 * (rms + n ** 0.5 + w.abs().amax() + 4)
        bad = ~((grads[k].double() - w).abs() <= tol)
        assert not bad.any(), (k, int(bad.sum()), grads[k][bad][:3].tolist(), w[bad][:3].tolist())


def test_join_is_the_join_of_the_dropped_output():
    """Without a norm after the block, bit for bit what dropout and the step make one after the other in 32 bits."""
    from bitsparse_amd.dropout import Dropout, dropout
    from bitsparse_amd.residual import block_join
    x, y = torch.randn(300, 520, device="cuda").requires_grad_(), torch.randn(300, 520, device="cuda").requires_grad_()
    drop = Dropout(0.25, 4, 5)                  # (its scale 4 / 3 rounds)
    a, b = block_join(x, y, drop=drop), block_join(x, dropout(y, drop))
    assert torch.equal(a, b)
    g = torch.randn_like(a)
    for i, j in zip(torch.autograd.grad(a, (x, y), g), torch.autograd.grad(b, (x, y), g)):
        assert torch.equal(i, j)


def test_join_dropped_values_pass_nothing():
    from bitsparse_amd.dropout import Dropout
    from bitsparse_amd.residual import block_join
    T, D = 40, 64
    m = torch.from_numpy(kept(range(T), D, 32768, 1, 2)).cuda()
    x, y = torch.randn(T, D, device="cuda"), torch.randn(T, D, device="cuda")
    y[~m] = torch.inf
    y[~m & (torch.rand(T, D, device="cuda") < 0.5)] = torch.nan
    gate = torch.rand(D, device="cuda").requires_grad_()
    y.requires_grad_()
    out = block_join(x, y, gate=gate, drop=Dropout(0.5, 1, 2))
    assert torch.equal(out[~m], x[~m]) and torch.isfinite(out).all()
    dy, dg = torch.autograd.grad(out, (y, gate), torch.ones_like(out))
    assert torch.isfinite(dy).all() and torch.isfinite(dg).all() and (dy[~m] == 0).all()


def test_join_state_and_graph_replays():
    """A captured step draws anew at each replay as its state moves on, the backward with its own forward."""
    from bitsparse_amd.dropout import Dropout, dropout
    from bitsparse_amd.residual import RowNorm, block_join
    T, D = 128, 256
    state = torch.tensor([7, 0], device="cuda")
    x, y = torch.randn(T, D, device="cuda").to(BF), torch.randn(T, D, device="cuda").to(BF)
    w = torch.ones(D, device="cuda").to(BF)
    gx, gh = torch.randn(T, D, device="cuda").to(BF), torch.randn(T, D, device="cuda").to(BF)
    one = torch.tensor([0, 1], device="cuda")

    def step(drop, x, y):
        x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
        d = dropout(y, drop)
        x1, h = block_join(x, d, pre=RowNorm(w), drop=drop)
        return x1, h, *torch.autograd.grad((x1, h), (x, y), (gx, gh))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(Dropout(0.4, state), x, y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(Dropout(0.4, state), x, y)
        state.add_(one)
    state.copy_(torch.tensor([7, 0]))
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(Dropout(0.4, 7, i), x, y)):
            assert torch.equal(a, b), i
