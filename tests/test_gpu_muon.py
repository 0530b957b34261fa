"""Orthogonalised updates (bitsparse_amd.muon) against the iteration in 64 bits.

Bars.  The kernels hold X, A and B as fp16 between products whose sums are
fp32; ``_model`` makes the same roundings in plain torch (fp32 products), so
its distance from the 64-bit iteration is what the format costs on that very
input, whatever the input's spectrum raises it to.  The kernels' own distance
may be a quarter more (the roundings fall otherwise where sums differ in
their last bits) plus 2e-4 of the result, a tenth of its rounding to bf16.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
COEF = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def _mod():
    from bitsparse_amd import muon
    return muon


def _exact(U, steps=5, coef=COEF, eps=EPS):
    """[B, R, C] in 64 bits"""
    U = U.double()
    tall = U.shape[-2] > U.shape[-1]
    X = U.mT.contiguous() if tall else U
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    a, b, c = coef
    for _ in range(steps):
        A = X @ X.mT.contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT.contiguous() if tall else X


def _model(U, steps=5, coef=COEF, eps=EPS):
    """The same with the kernels' roundings"""
    def h(t):
        return (t * 4096.0).half().float() / 4096.0
    tall = U.shape[-2] > U.shape[-1]
    X = U.double().mT.contiguous() if tall else U.double()
    X = h((X / (X.square().sum((-2, -1), keepdim=True).sqrt() + eps)).float())
    a, b, c = coef
    eye = torch.eye(X.shape[-2], device=X.device)
    for _ in range(steps):
        A = h(X @ X.mT.contiguous())
        X = h(h(a * eye + b * A + c * (A @ A)) @ X)
    return X.mT.contiguous() if tall else X


def _err(got, want):
    """2-norm of the difference over that of the result, the worst matrix of a batch"""
    return ((got.double() - want).square().sum((-2, -1)).sqrt() / want.square().sum((-2, -1)).sqrt().clamp(min=1e-30)).max().item()


def _grads(B, R, C, seed=0, kind="normal"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if kind == "normal":
        return rn(B, R, C)
    if kind == "low":       # fewer tokens than rows
        k = max(1, min(R, C) // 16)
        return rn(B, R, k) @ rn(B, k, C)
    if kind == "one":       # one token
        return rn(B, R, 1) @ rn(B, 1, C)
    m = min(R, C)           # singular values over four decades
    u, v = (torch.linalg.qr(rn(B, n, m))[0] for n in (R, C))
    return u * torch.logspace(0, -4, m, device="cuda") @ v.mT.contiguous()


def _check(U, got, **kw):
    U3 = U.reshape(-1, *U.shape[-2:])
    want = _exact(U3, **kw)
    model = _err(_model(U3, **kw).to(BF), want)
    assert got.dtype == BF and got.shape == U.shape and got.is_contiguous()
    err = _err(got.reshape(U3.shape), want)
    assert err <= 1.25 * model + 2e-4, (err, model)
    return err


SIZES = [(1, 1), (1, 5), (9, 1), (7, 3), (16, 48), (64, 64), (65, 130), (130, 65), (100, 1000), (256, 1024), (1024, 256),
         (513, 513), (1001, 333), (300, 5000), (768, 768), (1300, 2050)]


@pytest.mark.parametrize("R,C", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_sizes(R, C, dtype):
    G = _grads(1, R, C)[0].to(dtype)
    _check(G, _mod().orthogonalize(G))


@pytest.mark.parametrize("kind", ["low", "one", "decay"])
@pytest.mark.parametrize("R,C", [(96, 200), (700, 500), (512, 1024)])
def test_spectra(kind, R, C):
    G = _grads(1, R, C, 1, kind)[0]
    _check(G, _mod().orthogonalize(G))


def test_large():
    """More tiles than compute units, in each product."""
    G = _grads(1, 4096, 8200, 5)[0].to(BF)
    _check(G, _mod().orthogonalize(G))


@pytest.mark.parametrize("B,R,C", [(3, 70, 190), (5, 300, 128), (70, 33, 65), (24, 256, 300)])
def test_batches(B, R, C):
    G = _grads(B, R, C, 2)
    got = _mod().orthogonalize(G)
    _check(G, got)
    for i in (0, B - 1):        # a matrix's result does not depend on its company beyond the tile that is chosen
        assert _err(_mod().orthogonalize(G[i])[None], got[i][None].double()) < 4e-3


@pytest.mark.parametrize("steps,coef", [(1, COEF), (3, COEF), (12, (1.5, -0.5, 0.0)), (10, COEF)])
def test_steps_and_coefficients(steps, coef):
    G = _grads(1, 120, 250, 3)[0]
    _check(G, _mod().orthogonalize(G, steps=steps, coefficients=coef), steps=steps, coef=coef)


def test_singular_values():
    """What the operator is for: all of them near 1."""
    G = _grads(1, 200, 333, 4)[0]
    s = torch.linalg.svdvals(_mod().orthogonalize(G).float())
    assert s.max() < 1.25 and s.min() > 0.6
    # one token's gradient keeps its direction
    G = _grads(1, 200, 333, 4, "one")[0]
    O = _mod().orthogonalize(G).double()
    assert ((O * G).sum() / G.double().norm()).item() == pytest.approx((_exact(G[None])[0] * G).sum().item() / G.double().norm().item(), rel=4e-3)


def test_magnitudes_and_special_values():
    M = _mod()
    G = _grads(1, 60, 90, 6)[0]
    for scale in (2.0 ** 100, 2.0 ** -10):
        _check(G * scale, M.orthogonalize(G * scale))
    assert _check(G * 1e-9, M.orthogonalize(G * 1e-9)) < 1e-2       # eps counts: ||G|| = 7e-8
    assert not M.orthogonalize(torch.zeros(40, 70, device="cuda")).any()
    for bad in (math.inf, math.nan):
        H = G.clone()
        H[3, 4] = bad
        assert M.orthogonalize(H).isnan().all()
    assert M.orthogonalize(torch.zeros(0, 3, 4, device="cuda")).shape == (0, 3, 4)


def test_views():
    M = _mod()
    g = torch.Generator(device="cuda").manual_seed(7)
    big = torch.randn(4, 120, 303, generator=g, device="cuda").to(BF)
    for view in (big[:, 3:100, 5:205], big.transpose(0, 1)[1:101, :, 7:250].transpose(0, 1), big.mT, big[0], big[1].T,
                 big[:1, :, :50].expand(3, 120, 50)):
        assert torch.equal(M.orthogonalize(view), M.orthogonalize(view.contiguous()))
    four = big.reshape(2, 2, 120, 303)
    assert torch.equal(M.orthogonalize(four), M.orthogonalize(big).reshape(four.shape))


def _reference_update(W, G, M, lr, mu, nesterov, decay, s, steps=5):
    """(W', M') in 64 bits from the momentum as its type holds it, and the step's own error scale"""
    new = (mu * M.double() + (1 - mu) * G.double())
    stored = new.to(M.dtype)
    U = (1 - mu) * G.double() + mu * stored.double() if nesterov else stored.double()
    O = _exact(U[None])[0]
    noise = _err(_model(U.float()[None]), O[None])
    return (1 - lr * decay) * W.double() - lr * s * O, new, lr * s * O.norm().item() * (1.25 * noise + 5e-4)


@pytest.mark.parametrize("w,g,m", [(BF, BF, F32), (F32, F32, BF), (F32, BF, F32), (BF, F32, BF)])
@pytest.mark.parametrize("nesterov,decay,adjust", [(True, 0.1, "rms"), (False, 0.0, "shape"), (True, 0.0, 0.5)])
def test_update(w, g, m, nesterov, decay, adjust):
    """Shapes of both orientations, some of them together, odd ones, one of a single row."""
    mu, lr = 0.9, 0.05
    shapes = [(200, 80), (80, 200), (80, 200), (129, 129), (1, 77), (333, 1000)]
    W, G, M = ([_grads(1, *s, seed=10 * k + i)[0].to(t) * f for i, s in enumerate(shapes)]
               for k, (t, f) in enumerate([(w, 0.1), (g, 0.01), (m, 0.01)]))
    want = [_reference_update(*x, lr, mu, nesterov, decay,
                              0.2 * math.sqrt(max(s)) if adjust == "rms" else math.sqrt(max(1, s[0] / s[1])) if adjust == "shape" else adjust)
            for x, s in zip(zip(W, G, M), shapes)]
    versions = [t._version for t in W + M]
    _mod().muon_update_(W, G, M, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, adjust=adjust)
    assert all(t._version > v for t, v in zip(W + M, versions))
    for Wi, Mi, (ww, mm, noise) in zip(W, M, want):
        half = 2.0 ** -8 if Mi.dtype == BF else 2.0 ** -23      # (two products and a sum in fp32)
        assert ((Mi.double() - mm).abs() <= half * mm.abs() + 2.0 ** -23 * 0.05).all()
        half = 2.0 ** -8 if Wi.dtype == BF else 2.0 ** -23
        assert (Wi.double() - ww).norm() <= noise + half * ww.norm()


def test_update_in_place_of_views():
    """Weights inside a larger buffer: its other elements stay."""
    M = _mod()
    buf = torch.randn(100, 300, device="cuda")
    before = buf.clone()
    W, G, mom = buf[10:60, 7:140], torch.randn(133, 50, device="cuda").T, torch.zeros(50, 200, device="cuda")[:, :133]
    plain = W.clone()
    M.muon_update_([plain], [G.contiguous()], [mom.clone()], lr=0.1)
    M.muon_update_([W], [G], [mom], lr=0.1)
    assert torch.equal(W, plain)
    changed = buf != before
    # (an update of less than half a unit of its weight's last place leaves the weight as it is)
    step = torch.zeros_like(plain)
    M.muon_update_([step], [G.contiguous()], [torch.zeros(50, 133, device="cuda")], lr=0.1)
    lost = step.abs() <= before[10:60, 7:140].abs() * 2.0 ** -24
    assert (changed[10:60, 7:140] | lost).all() and lost.sum() < 10
    changed[10:60, 7:140] = False
    assert not changed.any()


def test_same_bits_streams_and_graph():
    M = _mod()
    G = _grads(2, 300, 700, 8).to(BF)
    first = M.orthogonalize(G)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = M.orthogonalize(G)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, other) and torch.equal(first, M.orthogonalize(G))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = M.orthogonalize(G)
    for i in range(4):
        G.copy_(_grads(2, 300, 700, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, M.orthogonalize(G))


def test_optimiser():
    """Training steps of a small block; the state saved and loaded again continues with the same bits."""
    from bitsparse_amd.bitsparse import TensorBuffer
    from bitsparse_amd.layers import FFNRelu2
    M = _mod()
    g = torch.Generator(device="cuda").manual_seed(9)
    W1 = (0.1 * torch.randn(256, 64, generator=g, device="cuda")).to(BF).requires_grad_()
    W2 = (0.1 * torch.randn(64, 256, generator=g, device="cuda")).to(BF).requires_grad_()
    x, target = (torch.randn(128, 64, generator=g, device="cuda").to(BF) for _ in range(2))
    buf = TensorBuffer(2 * 128 * 256, device="cuda")

    def steps(opt, W1, W2, n):
        losses = []
        for _ in range(n):
            buf.reset_buffer()
            loss = (FFNRelu2.apply(x, W1, W2, sparse_data=buf).float() - target.float()).square().mean()
            loss.backward()
            opt.step()
            opt.zero_grad()
            losses.append(loss.item())
        return losses
    opt = M.Muon([W1, W2], lr=0.02)
    losses = steps(opt, W1, W2, 20)
    assert losses[-1] < 0.8 * losses[0]
    V1, V2 = (w.detach().clone().requires_grad_() for w in (W1, W2))
    opt2 = M.Muon([V1, V2], lr=0.5)
    opt2.load_state_dict(opt.state_dict())
    assert steps(opt, W1, W2, 3) == steps(opt2, V1, V2, 3)
    assert torch.equal(W1, V1) and torch.equal(W2, V2)


def test_refusals():
    M = _mod()
    G = torch.randn(8, 12, device="cuda")
    for bad, kw, error in [(G[0], {}, ValueError), (G.half(), {}, TypeError), (G.cpu(), {}, RuntimeError),
                           (G, {"steps": 0}, ValueError), (G, {"steps": 101}, ValueError),
                           (torch.zeros(1, 65537, device="cuda"), {}, ValueError)]:
        with pytest.raises(error):
            M.orthogonalize(bad, **kw)
    W, m = torch.randn(8, 12, device="cuda"), torch.zeros(8, 12, device="cuda")
    for args, kw, error in [
            (([W], [G], []), {}, ValueError), (([W], [G.T.contiguous()], [m]), {}, ValueError), (([W.half()], [G], [m]), {}, TypeError),
            (([W], [G], [m.cpu()]), {}, RuntimeError), (([W.T], [G.T], [m.T]), {}, ValueError), (([W, W], [G, G], [m, m.clone()]), {}, ValueError),
            (([W[None]], [G[None]], [m[None]]), {}, ValueError), (([W], [G], [W]), {}, ValueError),
            (([W], [G], [m]), {"adjust": "adam"}, ValueError), (([W], [G], [m]), {"momentum": 1.0}, ValueError),
            (([W], [G], [m]), {"lr": -1.0}, ValueError), (([W], [G], [m]), {"steps": 0}, ValueError),
            (([W, W.clone()], [G, G], [m, m[:4]]), {}, ValueError)]:
        before = W.clone()
        with pytest.raises(error):
            M.muon_update_(*args, **{"lr": 0.1, **kw})
        assert torch.equal(W, before) and not m.any()
    M.muon_update_([], [], [], lr=0.1)
    with pytest.raises(ValueError):
        M.Muon([torch.nn.Parameter(torch.zeros(3, device="cuda"))])


# ---------------------------------------------------------------------------
# operands of 22 bits
# ---------------------------------------------------------------------------
def _model22(U, steps=5):
    """The iteration with the roundings of the precise form: each operand a sum of two fp16 numbers, products exact to
    fp32's sums but for low x low"""
    def h(t):
        hi = (t * 4096.0).half().float()
        return hi / 4096.0, (t * 4096.0 - hi).half().float() / 4096.0

    def mul(p, q):
        return p[0] @ q[0] + p[0] @ q[1] + p[1] @ q[0]
    X = U.double()
    X = h((X / (X.square().sum((-2, -1), keepdim=True).sqrt() + EPS)).float())
    a, b, c = COEF
    eye = torch.eye(U.shape[-2], device=U.device)
    for _ in range(steps):
        A = h(mul(X, tuple(x.mT.contiguous() for x in X)))
        B = h(a * eye + b * (A[0] + A[1]) + c * mul(A, A))
        Y = mul(B, X)
        X = h(Y)
    return Y


@pytest.mark.parametrize("kind", ["normal", "low", "one", "decay"])
@pytest.mark.parametrize("R,C", [(1, 3), (33, 100), (130, 260), (700, 500), (513, 2050)])
def test_precise(kind, R, C):
    """Into fp32 weights of 0: all that is left of them is the orthogonalised gradient.  The model's own sums are fp32 in
    another order than the kernels', and what they lose (some 2^-24 of a sum's terms) is raised like the operands'
    roundings: bar twice the model's distance, plus 2^-20."""
    G = _grads(1, R, C, 12, kind)[0]
    W, m = torch.zeros(R, C, device="cuda"), torch.zeros(R, C, device="cuda")
    _mod().muon_update_([W], [G], [m], lr=1.0, momentum=0.0, adjust=1.0)
    wide = G if R <= C else G.T.contiguous()
    want = _exact(wide[None])
    model = _err(_model22(wide[None]), want)
    got = -(W if R <= C else W.T)
    err = _err(got[None], want)
    assert err <= 2 * model + 2.0 ** -20, (err, model)
    # in bf16: nothing but the result's own rounding is left, half a unit
    O = _mod().orthogonalize(wide, precise=True)
    tol = 2.0 ** -8 * want[0].abs() + 2 * (2 * model + 2.0 ** -20) * want[0].norm()
    assert ((O.double() - want[0]).abs() <= tol).all()


def test_precise_or_not():
    """fp32 weights are precise unless told otherwise, bf16 ones the other way round; either may choose."""
    G, m = _grads(1, 200, 300, 13)[0], torch.zeros(200, 300, device="cuda")
    want = _exact(G[None])
    errs = {}
    for dtype in (F32, BF):
        for precise in (None, True, False):
            W = torch.zeros(200, 300, device="cuda", dtype=dtype)
            _mod().muon_update_([W], [G], [m.clone()], lr=1.0, momentum=0.0, adjust=1.0, precise=precise)
            errs[dtype, precise] = _err(-W[None], want)
    assert errs[F32, None] == errs[F32, True] < 1e-5 and 5e-4 < errs[F32, False] < 3e-3
    assert errs[BF, None] == errs[BF, False] > errs[BF, True]


@pytest.mark.parametrize("B,R,C", [(1, 2304, 4700), (3, 1000, 3100), (2, 1024, 4100), (65, 200, 70)])
@pytest.mark.parametrize("precise", [False, True])
def test_shared_tiles(B, R, C, precise):
    """Counts of tiles that leave a last round to be dealt out in shares, several matrices of them; more matrices than
    go together."""
    G = _grads(B, R, C, 14).to(BF)
    got = _mod().orthogonalize(G, precise=precise)
    if precise:
        assert _err(got, _exact(G)) < 2.0e-3
    else:
        _check(G, got)


@pytest.mark.parametrize("B,R,C", [(1, 64, 8200), (3, 200, 9000), (2, 130, 600), (70, 48, 100), (5, 256, 256), (1, 16000, 190)])
@pytest.mark.parametrize("precise", [False, True])
def test_few_rows(B, R, C, precise):
    """Up to 256 rows, whose polynomial is not formed; long K, which is split over workgroups; the bars of the other
    shapes."""
    G = _grads(B, R, C, 15).to(BF)
    got = _mod().orthogonalize(G, precise=precise)
    if precise:
        assert _err(got, _exact(G)) < 2.0e-3
    else:
        _check(G, got)
    assert torch.equal(got, _mod().orthogonalize(G, precise=precise))
