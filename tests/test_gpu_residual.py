"""The step between two blocks (bitsparse_amd.residual) against its formulas
in 64 bits.

Bars, from the number formats.  A result is rounded once, so it is within
half a unit (2^-8 of its value at most in bf16, 2^-24 in fp32) of what the kernel's
32-bit arithmetic gives; that in turn is off by a few roundings of 2^-24 in
each term of its sums, bounded here by 2^-19 of the sum of the terms'
magnitudes (32 roundings; the longest chain of additions, 32768 elements over
up to 1024 lanes, has 32 in a lane, 6 in a wave and 16 over waves, and
roundings of random sign add up to far less than their count).  x' is checked
first and the rest is compared with what follows from x' as stored.
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def _mod():
    from bitsparse_amd import residual
    return residual


def _std(v, kind):
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1 / ((c * c).mean(-1, keepdim=True) + EPS).sqrt()
    return c * r, r


def _std_grad(dn, n, r, kind):
    """(gradient, bound on the sum of its terms' magnitudes)"""
    m0 = dn.mean(-1, keepdim=True) if kind == "layer" else 0.0
    m1 = (dn * n).mean(-1, keepdim=True)
    mag = r * (dn.abs() + dn.abs().mean(-1, keepdim=True) + n.abs() * (dn * n).abs().mean(-1, keepdim=True))
    return r * (dn - m0 - n * m1), mag


def _close(got, want, mag, name):
    want, mag = want.reshape(got.shape), mag.expand_as(want).reshape(got.shape)
    half = 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    tol = half * want.abs() * (1 + 2.0 ** -6) + 2.0 ** -19 * mag + 1e-37
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3].tolist(), want[bad][:3].tolist())


def _inputs(T, D, xt, yt, gate, scale, bias, vt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    t = {"x": (rn(T, D) * 2 + rn(D)).to(xt), "y": (rn(T, D) + 0.5 * rn(D)).to(yt),
         "w_post": (1 + 0.2 * rn(D)).to(vt), "w_pre": (1 + 0.2 * rn(D)).to(vt),
         "b_post": (0.1 * rn(D)).to(vt) if bias else None, "b_pre": (0.1 * rn(D)).to(vt) if bias else None,
         "gate": None, "scale": None}
    shape = {"one": (1,), "channel": (D,), "row": (T, 1), "element": (T, D)}
    if gate is not None:
        t["gate"] = (0.5 + 0.3 * rn(*shape[gate])).to(yt if gate == "element" else vt)
    if scale in shape:
        t["scale"] = (0.9 + 0.1 * rn(*shape[scale])).to(vt)
    return t, rn(T, D).to(xt), rn(T, D).to(yt)


def _reference(t, x1, g_x, g_h, post, pre, scale_value):
    """Expected results and the magnitudes of their sums' terms; x1: x' as the kernel stored it."""
    v = {k: None if p is None else p.detach().double() for k, p in t.items()}
    one = torch.ones((), dtype=torch.float64, device="cuda")
    gate = one if v["gate"] is None else v["gate"]
    s = one * scale_value if v["scale"] is None else v["scale"]
    w1 = one if v["w_post"] is None or not post else v["w_post"]
    b1 = one * 0 if v["b_post"] is None or not post else v["b_post"]
    yn, yr = _std(v["y"], post) if post else (v["y"], one)
    p = yn * w1 + b1
    # (a layer norm subtracts numbers of the row's size)
    ymag = (v["y"].abs() + v["y"].abs().mean(-1, keepdim=True)) * yr
    out = {"x1": (s * v["x"] + gate * p, (s * v["x"]).abs() + (gate * w1).abs() * ymag + (gate * b1).abs())}
    G, Gm = (g_x.double(), g_x.double().abs()) if g_x is not None else (one * 0, one * 0)
    if pre:
        w2 = one if v["w_pre"] is None else v["w_pre"]
        xn, xr = _std(x1.double(), pre)
        xmag = (x1.double().abs() + x1.double().abs().mean(-1, keepdim=True)) * xr
        out["h"] = (xn * w2 + (0 if v["b_pre"] is None else v["b_pre"]), w2.abs() * xmag + (0 if v["b_pre"] is None else v["b_pre"].abs()))
        if g_h is not None:
            gh = g_h.double()
            out["dw_pre"] = ((gh * xn).sum(0), (gh.abs() * xmag).sum(0))
            out["db_pre"] = (gh.sum(0), gh.abs().sum(0))
            d, m = _std_grad(gh * w2, xn, xr, pre)
            G, Gm = G + d, Gm + m + (d.abs() * 4 * xmag.amax(-1, keepdim=True).clamp(max=16))
    G, Gm = G.expand_as(v["x"]), Gm.expand_as(v["x"])
    out["dx"] = (s * G, s.abs() * Gm)
    ds, dsm = G * v["x"], Gm * v["x"].abs()
    out["dscale"] = (ds.sum(0), dsm.sum(0)) if v["scale"] is None or v["scale"].numel() > 1 or ds.shape[1] == 1 else (ds.sum().reshape(1), dsm.sum().reshape(1))
    pm = w1.abs() * ymag + b1.abs()
    dg, dgm = G * p, Gm * pm
    if v["gate"] is not None:
        for d in range(dg.dim()):
            if v["gate"].dim() == 1 and d == 0 or v["gate"].dim() == 2 and v["gate"].shape[d] == 1:
                dg, dgm = dg.sum(d, keepdim=True), dgm.sum(d, keepdim=True)
        if v["gate"].numel() == 1:
            dg, dgm = dg.sum().reshape(1), dgm.sum().reshape(1)
    out["dgate"] = (dg, dgm)
    dp, dpm = gate * G, gate.abs() * Gm
    out["dw_post"] = ((dp * yn).sum(0), (dpm * ymag).sum(0))
    out["db_post"] = (dp.sum(0), dpm.sum(0))
    if post:
        d, m = _std_grad(dp * w1, yn, yr, post)
        m2 = yr * (w1.abs() * dpm + (w1.abs() * dpm).mean(-1, keepdim=True) + ymag * (w1.abs() * dpm * ymag).mean(-1, keepdim=True))
        out["dy"] = (d, m + m2)
    else:
        out["dy"] = (dp, dpm)
    return out


def _check(T, D, xt=BF, yt=BF, post="rms", pre="rms", gate="channel", scale="channel", bias=False, vt=F32, use=("x", "h"), seed=0):
    R = _mod()
    t, g_x, g_h = _inputs(T, D, xt, yt, gate, scale, bias, vt, seed)
    if not post:
        t["w_post"] = t["b_post"] = None
    if not pre:
        t["w_pre"] = t["b_pre"] = None
    leaves = {k: p.requires_grad_() for k, p in t.items() if p is not None}
    value = scale if isinstance(scale, float) else 1.0
    out = R.block_join(t["x"], t["y"], post=R.RowNorm(t["w_post"], t["b_post"], post, EPS) if post else None, gate=t["gate"],
                       scale=t["scale"] if t["scale"] is not None else scale,
                       pre=R.RowNorm(t["w_pre"], t["b_pre"], pre, EPS) if pre else None)
    x1, h = out if pre else (out, None)
    assert x1.dtype == xt and x1.shape == (T, D) and (h is None or h.dtype == yt)
    ends, seeds = [], []
    if "x" in use:
        ends, seeds = ends + [x1], seeds + [g_x]
    if "h" in use and pre:
        ends, seeds = ends + [h], seeds + [g_h]
    grads = dict(zip(leaves, torch.autograd.grad(ends, list(leaves.values()), seeds, allow_unused=True)))
    want = _reference(t, x1.detach(), g_x if "x" in use else None, g_h if "h" in use and pre else None, post, pre, value)
    _close(x1.detach(), *want["x1"], "x1")
    if pre:
        _close(h.detach(), *want["h"], "h")
    for k, g in grads.items():
        if "d" + k not in want:                 # (the next norm's vectors without a gradient of h)
            assert g is None or not g.any(), k
            continue
        assert g.dtype == t[k].dtype and g.shape == t[k].shape
        _close(g, *want["d" + k], "d" + k)


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (4, 511), (9, 512), (2, 513), (7, 1000), (5, 1024), (3, 1025), (130, 96), (2, 1536),
         (6, 2501), (2, 4096), (3, 4097), (2, 8191), (2, 8192), (2, 8200), (2, 16384), (2, 16389), (1, 32768), (1500, 320),
         (1031, 1032), (2100, 72)]


@pytest.mark.parametrize("T,D", SIZES)
@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (F32, F32)])
def test_sizes(T, D, xt, yt):
    _check(T, D, xt, yt, post="layer", pre="rms", bias=True)
    _check(T, D, xt, yt, post="rms", pre="layer", bias=False, vt=xt, gate="row", scale="one")


@pytest.mark.parametrize("gate,scale", itertools.product([None, "one", "channel", "row", "element"], [None, 0.5, "one", "channel"]))
@pytest.mark.parametrize("T,D", [(37, 200), (11, 1300)])
def test_gates_and_scales(gate, scale, T, D):
    _check(T, D, gate=gate, scale=scale, bias=True, post="layer", pre="layer")
    _check(T, D, F32, BF, gate=gate, scale=scale, post="rms", pre="rms", vt=BF)


@pytest.mark.parametrize("post,pre,use", [(None, "rms", "xh"), ("rms", None, "x"), (None, None, "x"), ("layer", "layer", "h"),
                                          ("layer", "layer", "x"), (None, "layer", "h")])
@pytest.mark.parametrize("gate", [None, "channel", "row", "element"])
def test_parts(post, pre, use, gate):
    for T, D in ((21, 129), (9, 1801)):
        _check(T, D, post=post, pre=pre, use=use, gate=gate, bias=True)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("T,D", [(1, 4096), (40, 77), (700, 768), (3, 9000)])
@pytest.mark.parametrize("xt,ht", [(BF, BF), (F32, BF), (F32, F32)])
def test_norm_alone(kind, T, D, xt, ht):
    R = _mod()
    t, _, g_h = _inputs(T, D, xt, ht, None, None, True, F32)
    x, w, b = (t[k].requires_grad_() for k in ("x", "w_pre", "b_pre"))
    h = R.block_norm(x, R.RowNorm(w, b, kind, EPS), dtype=ht)
    assert h.dtype == ht
    want = _reference({**t, "w_post": None, "b_post": None}, x.detach(), None, g_h, None, kind, 1.0)
    _close(h.detach(), *want["h"], "h")
    dx, dw, db = torch.autograd.grad(h, (x, w, b), g_h)
    _close(dx, *want["dx"], "dx")
    _close(dw, *want["dw_pre"], "dw")
    _close(db, *want["db_pre"], "db")
    with torch.no_grad():
        assert torch.equal(R.block_norm(x, R.RowNorm(w, b, kind, EPS), dtype=ht), h)


def test_gradients_against_differences():
    """d/de of <g, outputs> along random directions of every operand, by central differences of the kernel's own
    forward in fp32.  The step e moves an operand by 2^-6 of its values: the quotient's own error is e^2 times
    third derivatives (under 1e-3 of the result here) and 2^-24 / e of roundings that average out over 4000 results."""
    R = _mod()
    t, g_x, g_h = _inputs(40, 100, F32, F32, "channel", "channel", True, F32)

    def loss(t):
        x1, h = R.block_join(t["x"], t["y"], post=R.RowNorm(t["w_post"], t["b_post"], "layer", EPS), gate=t["gate"],
                             scale=t["scale"], pre=R.RowNorm(t["w_pre"], t["b_pre"], "layer", EPS))
        return x1, h
    leaves = {k: p.clone().requires_grad_() for k, p in t.items()}
    grads = torch.autograd.grad(loss(leaves), list(leaves.values()), (g_x, g_h))
    for k, g in zip(leaves, grads):
        d = g / g.norm() + 0.1 * torch.randn_like(g) / math.sqrt(g.numel())     # mostly along the gradient: no cancelled sum
        e = 2.0 ** -6 * t[k].norm() / d.norm()
        a, b = (sum((o.double() * q.double()).sum() for o, q in zip(loss({**t, k: t[k] + s * e * d}), (g_x, g_h))) for s in (1, -1))
        got, want = (g.double() * d.double()).sum().item(), ((a - b) / (2 * e)).item()
        assert abs(got - want) < 5e-3 * abs(want), (k, got, want)


def test_strides_and_shapes():
    """Views: rows inside wider rows at odd addresses, a batch whose tokens are not contiguous, gradients that were
    expanded, vectors with a stride."""
    R = _mod()
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(6, 50, 403, generator=g, device="cuda").to(BF)
    wide = torch.randn(2, 260, generator=g, device="cuda")
    x, y = big[:, :, 3:133], big.transpose(0, 1)[:, :, 201:331].transpose(0, 1)
    gate, w = wide[0, ::2], wide[1, 1::2]
    pre = R.RowNorm(w, None, "layer", EPS)
    got = R.block_join(x, y, gate=gate, pre=pre)
    want = R.block_join(x.contiguous(), y.contiguous(), gate=gate.contiguous(), pre=R.RowNorm(w.contiguous(), None, "layer", EPS))
    assert all(torch.equal(a, b) and a.shape == x.shape for a, b in zip(got, want))
    # a batch of tokens cut out of a longer one: no single row stride
    part = big[:, 5:40, 8:138]
    assert torch.equal(R.block_norm(part, pre), R.block_norm(part.contiguous(), pre))
    grads = []
    for copy in (False, True):
        xs, ws = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        x1, h = R.block_join(xs, y, gate=gate, pre=R.RowNorm(ws, None, "layer", EPS))
        seed = torch.full((1, 1, 1), 0.5, dtype=BF, device="cuda").expand(x.shape)
        grads.append(torch.autograd.grad((x1, h), (xs, ws), (seed.contiguous(), seed.contiguous()) if copy else (seed, seed)))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    v = torch.randn(130, generator=g, device="cuda").to(BF)
    assert torch.equal(R.block_norm(v, pre), R.block_norm(v[None], pre)[0])


def test_no_rows():
    R = _mod()
    x, w = torch.zeros(0, 5, 64, device="cuda", dtype=BF, requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    x1, h = R.block_join(x, x, gate=w, pre=R.RowNorm(w))
    assert x1.shape == h.shape == (0, 5, 64)
    gx, gw = torch.autograd.grad((x1, h), (x, w), (torch.zeros_like(x1), torch.zeros_like(h)))
    assert gx.shape == x.shape and not gw.any()


@pytest.mark.parametrize("D", [64, 2000])
def test_special_rows(D):
    """A row of zeros, of one huge value, with an infinity, with a NaN: each stays in its own row."""
    R = _mod()
    x = torch.randn(6, D, device="cuda")
    x[0] = 0
    x[1] = 0
    x[1, 3] = 2.0 ** 60
    x[2, 5] = math.inf
    x[3, 7] = math.nan
    x[4] = 1000.0 + 2.0 ** -6 * torch.randn(D, device="cuda")       # a mean far above the deviations
    for kind in ("rms", "layer"):
        h = R.block_norm(x, R.RowNorm(None, None, kind, EPS))
        assert not h[0].any()
        assert torch.isfinite(h[1]).all()
        assert h[3].isnan().all() and (h[2].isnan() | (h[2] == 0)).all()
        want = _std(x[4:].double(), kind)[0]
        # (the deviations of the fifth row are known to 2^-24 of the values they come from)
        assert (h[4:].double() - want).abs().max() < (2.0 ** -24 * 1000 * 4 / 2.0 ** -6 if kind == "layer" else 1e-5)


def test_same_bits_and_streams():
    R = _mod()
    t, g_x, g_h = _inputs(3000, 600, BF, BF, "one", "one", True, F32)
    leaves = [t[k].requires_grad_() for k in ("x", "y", "w_post", "b_post", "w_pre", "b_pre", "gate", "scale")]

    def step():
        x1, h = R.block_join(t["x"], t["y"], post=R.RowNorm(t["w_post"], t["b_post"]), gate=t["gate"], scale=t["scale"],
                             pre=R.RowNorm(t["w_pre"], t["b_pre"]))
        return [x1, h, *torch.autograd.grad((x1, h), leaves, (g_x, g_h))]
    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b, c in zip(first, other, step()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replays():
    R = _mod()
    x, y = (torch.randn(64, 768, device="cuda").to(BF) for _ in range(2))
    w = torch.ones(768, device="cuda")
    run = lambda: R.block_join(x, y, post=R.RowNorm(w), pre=R.RowNorm(w, None, "layer"))  # noqa: E731
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for i in range(4):
            x.copy_(torch.randn(64, 768, device="cuda"))
            y.mul_(1.5)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, run()))


def test_past_32_bit_offsets():
    """2^31 + 2^21 elements and more, rows at both ends and in the middle."""
    R = _mod()
    T, D = 2 ** 19 + 512, 4100
    x = torch.empty(T, D, dtype=BF, device="cuda")
    rows = torch.tensor([0, 1, T // 2, 2 ** 31 // D, 2 ** 31 // D + 1, T - 2, T - 1], device="cuda")
    x.zero_()
    x[rows] = torch.randn(len(rows), D, device="cuda").to(BF)
    w = torch.rand(D, device="cuda").requires_grad_()
    x.requires_grad_()
    h = R.block_norm(x, R.RowNorm(w))
    few = x.detach()[rows].requires_grad_()
    w2 = w.detach().clone().requires_grad_()
    h2 = R.block_norm(few, R.RowNorm(w2))
    assert torch.equal(h.detach()[rows], h2.detach())
    g = torch.zeros_like(x)
    g[rows] = 1
    dx, dw = torch.autograd.grad(h, (x, w), g)
    dx2, dw2 = torch.autograd.grad(h2, (few, w2), torch.ones_like(few))
    assert torch.equal(dx[rows], dx2) and torch.allclose(dw, dw2, rtol=1e-5, atol=1e-5)


def test_refusals():
    R = _mod()
    x = torch.zeros(4, 64, device="cuda", dtype=BF)
    n = R.RowNorm()
    for args, kw, error in [
            ((x.half(), n), {}, TypeError), ((x, n), {"dtype": F32}, TypeError), ((x, n), {"dtype": torch.float16}, TypeError),
            ((x.cpu(), n), {}, RuntimeError), ((x, None), {}, TypeError), ((x, R.RowNorm(kind="batch")), {}, ValueError),
            ((x, R.RowNorm(eps=-1.0)), {}, ValueError), ((x, R.RowNorm(torch.ones(63, device="cuda"))), {}, ValueError),
            ((x, R.RowNorm(torch.ones(64))), {}, RuntimeError),
            ((x, R.RowNorm(torch.ones(64, device="cuda").half())), {}, TypeError),
            ((x[:, :0], n), {}, ValueError), ((torch.zeros(1, 32769, device="cuda"), n), {}, ValueError),
            ((torch.zeros((), device="cuda"), n), {}, ValueError)]:
        with pytest.raises(error):
            R.block_norm(*args, **kw)
    for args, kw, error in [
            ((x, x[:3]), {}, ValueError), ((x, x.float()), {}, TypeError), ((x, None), {}, TypeError),
            ((x, x), {"gate": torch.ones(4, 2, device="cuda")}, ValueError),
            ((x, x), {"gate": torch.ones(4, device="cuda")}, ValueError),
            ((x, x), {"scale": torch.ones(4, 1, device="cuda")}, ValueError)]:
        with pytest.raises(error):
            R.block_join(*args, **kw)
    xs = x.clone().requires_grad_()
    g, = torch.autograd.grad(R.block_norm(xs, n).sum(), xs)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(R.block_norm(xs, n).sum(), xs, create_graph=True)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.vmap(lambda r: R.block_norm(r, n))(x)


def test_partial_walks():
    """Gradients of some operands alone are those of a full walk."""
    R = _mod()
    t, g_x, g_h = _inputs(50, 300, BF, BF, "channel", "channel", True, F32)
    names = ("x", "y", "w_post", "b_post", "gate", "scale", "w_pre", "b_pre")
    leaves = [t[k].requires_grad_() for k in names]
    x1, h = R.block_join(t["x"], t["y"], post=R.RowNorm(t["w_post"], t["b_post"], "layer"), gate=t["gate"], scale=t["scale"],
                         pre=R.RowNorm(t["w_pre"], t["b_pre"], "layer"))
    full = torch.autograd.grad((x1, h), leaves, (g_x, g_h), retain_graph=True)
    for i, p in enumerate(leaves):
        one, = torch.autograd.grad((x1, h), p, (g_x, g_h), retain_graph=True)
        assert torch.equal(one, full[i]), names[i]
