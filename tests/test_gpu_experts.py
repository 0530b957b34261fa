"""Routing, the experts' products and the weighted sum (bitsparse_amd.experts) against their formulas in 64 bits.

Bars, from the number formats.  A result is rounded once: within half a unit,
2^-8 of its value in bf16 and 2^-24 in fp32, of what 32-bit arithmetic gives.
A 32-bit sum of n terms is off by less than n roundings of 2^-24 of the sum of
their magnitudes.  The gradient of gathered tokens is a sum of rows that are
rounded to bf16 by themselves first.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def _mod():
    from bitsparse_amd import experts
    return experts


def _close(got, want, mag, terms, name):
    tol = HALF[got.dtype] * want.abs() * (1 + 2.0 ** -6) + (terms + 4) * 2.0 ** -24 * mag + 1e-37
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3].tolist(), want[bad][:3].tolist())


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rn(g, *s):
    return torch.randn(s, generator=g, device="cuda")


def _ids(T, k, E, g, lost=0.0, skew=0.5):
    ids = (_rn(g, T, E) + skew * _rn(g, E)).topk(k, -1).indices.int()
    if lost:
        ids[torch.rand(T, k, generator=g, device="cuda") < lost] = -1
    return ids


def _plain_plan(ids, E):
    flat = ids.reshape(-1).tolist()
    order = sorted((i for i, e in enumerate(flat) if 0 <= e < E), key=lambda i: (flat[i], i))
    offsets = [sum(0 <= e < x for e in flat) for x in range(E)] + [len(order)]
    place = [-1] * len(flat)
    for r, i in enumerate(order):
        place[i] = r
    dev = ids.device
    return (torch.tensor(offsets, device=dev).int(), torch.tensor(order + [-1] * (len(flat) - len(order)), device=dev).int(),
            torch.tensor(place, device=dev).int().view(ids.shape))


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 64), (7, 3, 5), (64, 2, 1024), (257, 4, 3 + 4), (1000, 8, 96), (4097, 1, 8), (2500, 2, 1024), (70000, 2, 40)])
def test_plan(T, k, E):
    g = _gen(T + E)
    ids = torch.randint(-2, E + 2, (T, k), generator=g, device="cuda").int()
    for got, want in zip(_mod().plan_experts(ids, E), _plain_plan(ids, E)):
        assert torch.equal(got, want)


def test_plan_of_one_expert_and_of_none():
    m = _mod()
    for ids, E in ((torch.full((300, 2), 3), 7), (torch.full((300, 2), -1), 7), (torch.full((5, 1), 7), 7), (torch.zeros(0, 2), 4)):
        ids = ids.int().cuda()
        for got, want in zip(m.plan_experts(ids, E), _plain_plan(ids, E)):
            assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# route
# ---------------------------------------------------------------------------
def _route(l, k, score, bias, groups, top_groups, best, renorm, scale):
    """(weights, experts, s) in 64 bits"""
    l = l.double()
    T, E = l.shape
    s = torch.softmax(l, -1) if score == "softmax" else torch.sigmoid(l)
    c = s if bias is None else s + bias.double()
    c = torch.where(l == -torch.inf, -torch.inf, c)
    if top_groups < groups:
        by = c.view(T, groups, -1)
        keep = torch.sort(torch.sort(by, dim=-1, descending=True).values[..., :best].sum(-1), dim=-1, descending=True, stable=True).indices[:, :top_groups]
        mask = torch.zeros(T, groups, dtype=torch.bool, device=l.device).scatter_(1, keep, True)
        c = by.masked_fill(~mask[..., None], -torch.inf).view(T, E)
    top = torch.sort(c, dim=-1, descending=True, stable=True)
    ids = torch.where(top.values[:, :k] > -torch.inf, top.indices[:, :k], -1)
    w = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0)), 0.0)
    if renorm:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return w * scale, ids, s


ROUTES = [(1, 64, 8, "sigmoid", True, 8, 4, 2, True), (33, 8, 2, "softmax", False, 1, 1, 1, True), (5, 1, 1, "softmax", False, 1, 1, 1, False),
          (257, 257, 7, "softmax", True, 1, 1, 1, False), (64, 256, 8, "sigmoid", True, 8, 4, 2, True), (40, 1024, 64, "sigmoid", False, 64, 9, 1, False),
          (100, 60, 6, "softmax", True, 6, 3, 2, True), (9, 128, 3, "softmax", False, 4, 1, 1, True), (70, 5, 5, "sigmoid", False, 5, 5, 1, True),
          (31, 600, 20, "softmax", False, 1, 1, 1, True), (31, 12, 3, "sigmoid", True, 12, 3, 2, True)]


@pytest.mark.parametrize("T,E,k,score,bias,groups,top_groups,best,renorm", ROUTES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_route(T, E, k, score, bias, groups, top_groups, best, renorm, dtype):
    g = _gen(T + E)
    l = (_rn(g, T, 2 * E) * 1.5).to(dtype)[:, :E].requires_grad_()
    b = 0.1 * _rn(g, E) if bias else None
    w, ids = _mod().route(l, k, score=score, bias=b, groups=groups, top_groups=top_groups, group_best=best, renormalize=renorm, scale=1.7)
    want, want_ids, s = _route(l.detach(), k, score, b, groups, top_groups, best, renorm, 1.7)
    assert torch.equal(ids.long(), want_ids)
    assert ids.dtype == torch.int32 and w.dtype == F32 and not ids.requires_grad
    # (a softmax's is divided by a sum of E exponentials, which is off by less than E roundings)
    _close(w.detach(), want, want, E if score == "softmax" else 4, "w")
    dw = _rn(g, T, k)
    dl, = torch.autograd.grad(w, l, dw)
    # by the formulas; E + k terms of a token's sums, scores and exponentials a few roundings each
    at = ids.long()
    sc = s.gather(1, at)
    total = sc.sum(-1, keepdim=True) if renorm else torch.ones_like(sc[:, :1])
    gw = dw.double() * 1.7
    ds = (gw - (gw * sc).sum(-1, keepdim=True) / total) / total if renorm else gw
    mag = (gw.abs() + (gw * sc).abs().sum(-1, keepdim=True) / total) / total if renorm else gw.abs()
    full, full_mag = (torch.zeros_like(s).scatter_(1, at, v) for v in (ds, mag))
    if score == "softmax":
        want, want_mag = s * (full - (full * s).sum(-1, keepdim=True)), s * (full_mag + (full_mag * s).sum(-1, keepdim=True))
    else:
        want, want_mag = s * (1 - s) * full, s * full_mag
    _close(dl, want, want_mag, 2 * (E + k) + 32, "dlogits")


def test_route_gradient_against_differences():
    g = _gen(3)
    for score, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        l = _rn(g, 6, 16).requires_grad_()
        dw = _rn(g, 6, 4)
        w, ids = _mod().route(l, 4, score=score, renormalize=renorm)
        dl, = torch.autograd.grad(w, l, dw)
        d = _rn(g, 6, 16).double()
        h = 1e-5

        def f(x):
            s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
            v = s.gather(1, ids.long())
            return ((v / v.sum(-1, keepdim=True) if renorm else v) * dw.double()).sum()
        x = l.detach().double()
        slope = (f(x + h * d) - f(x - h * d)) / (2 * h)
        # central differences: h^2 of a third derivative of order one, and 2^-52 / h
        assert abs(slope - (dl.double() * d).sum()) < 1e-6 * (1 + dl.abs().sum().item())


def test_route_ties_go_by_index():
    m = _mod()
    l = torch.zeros(3, 70, device="cuda")
    for score in ("softmax", "sigmoid"):
        w, ids = m.route(l, 5, score=score)
        assert torch.equal(ids, torch.arange(5, device="cuda").int().expand(3, 5))
        # s / (s + s + s + s + s) in 32 bits: the sum is at most three times rounded (2 s is exact), the quotient once
        _close(w, torch.full_like(w, 0.2, dtype=torch.float64), 0.2, 3, "w")
        w, ids = m.route(l, 4, score=score, groups=7, top_groups=2, group_best=2, bias=torch.zeros(70, device="cuda"))
        assert torch.equal(ids, torch.arange(4, device="cuda").int().expand(3, 4))
    # next to each other in 32 bits, apart in 64
    l = torch.zeros(1, 8, device="cuda")
    l[0, 5] = 1e-9
    assert m.route(l, 1)[1].item() == 5 and m.route(l, 1, score="sigmoid")[1].item() == 5


@pytest.mark.parametrize("E,k,groups,top_groups,best", [(256, 8, 8, 4, 2), (64, 6, 1, 1, 1), (8, 2, 1, 1, 1), (300, 5, 1, 1, 1), (48, 4, 3, 2, 2), (128, 8, 8, 3, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_of_many_equal_and_close_values(E, k, groups, top_groups, best, score, biased):
    """Logits on a coarse grid, most of them equal to others, and some of them a few units of the last place beside: equal
    values by index, close ones by their order in 64 bits."""
    g = _gen(E + k)
    T = 3000
    l = (_rn(g, T, E) * 4).round() / 4
    close = torch.rand(T, E, generator=g, device="cuda") < 0.3
    l = torch.where(close, l * (1 + 2.0 ** -22 * torch.randint(-3, 4, (T, E), generator=g, device="cuda")), l)
    b = (_rn(g, E) * 4).round() / 64 if biased else None
    w, ids = _mod().route(l, k, score=score, bias=b, groups=groups, top_groups=top_groups, group_best=best)
    _, want, _ = _route(l, k, score, b, groups, top_groups, best, True, 1.0)
    # (what a bias is added to is rounded: where two of the reference's values are within 2^-50 its order may be its roundings')
    s = (torch.softmax if score == "softmax" else lambda v, d: torch.sigmoid(v))(l.double(), -1)
    c = s if b is None else s + b.double()
    differ = ids.long() != want
    gap = (c.gather(1, ids.long()) - c.gather(1, want)).abs()
    assert (gap[differ] < 2.0 ** -50).all(), (int(differ.sum()), gap[differ].max().item())
    assert differ.float().mean() < 0.01
    assert (ids.sort(-1).values.diff(dim=-1) > 0).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_groups_whose_best_cancel(score):
    """Biases that take a group's two best far apart on both sides of 0: the sums that decide are small and close together, the
    values that they are of are not."""
    g = _gen(17)
    T, E, groups = 4096, 64, 4
    l = 4e-5 * _rn(g, T, E)
    b = torch.full((E,), -torch.inf, device="cuda")
    b[::16], b[5::16] = 10.0, -10.0
    w, ids = _mod().route(l, 2, score=score, bias=b, groups=groups, top_groups=1, group_best=2)
    _, want, s = _route(l, 2, score, b, groups, 1, 2, True, 1.0)
    both = s[:, ::16] + s[:, 5::16]
    top = both.topk(2, -1).values
    sure = top[:, 0] - top[:, 1] > 2.0 ** -47           # (four roundings of 10 in 64 bits are 2^-49 each)
    assert sure.float().mean() > 0.99 and torch.equal(ids[sure].long(), want[sure])


def test_route_masked_logits():
    m = _mod()
    l = _rn(_gen(1), 6, 20)
    l[0] = -torch.inf                   # a padded token
    l[1, 3:] = -torch.inf               # fewer experts than choices
    l[2, 7] = torch.nan
    l[3, ::2] = -torch.inf
    for score in ("softmax", "sigmoid"):
        x = l.clone().requires_grad_()
        w, ids = m.route(x, 5, score=score)
        assert ids[0].tolist() == [-1] * 5 and w[0].tolist() == [0.0] * 5
        assert sorted(ids[1, :3].tolist()) == [0, 1, 2] and ids[1, 3:].tolist() == [-1, -1]
        assert abs(w[1].sum().item() - 1) < 1e-6
        assert w[2].isnan().any() and (0 <= ids[2]).all() and (ids[2] < 20).all()
        assert (ids[3] % 2 == 1).all()
        if score == "sigmoid":
            assert ids[2, 0] == 7
        dl, = torch.autograd.grad(w, x, torch.ones_like(w))
        keep = torch.tensor([0, 1, 3, 4, 5])
        assert torch.isfinite(dl[keep]).all() and (dl[0] == 0).all() and (dl[1, 3:] == 0).all()
    bias = torch.zeros(20, device="cuda")
    bias[4:] = -torch.inf
    w, ids = m.route(l[4:], 6, bias=bias, score="sigmoid")
    assert (ids[:, :4].sort().values == torch.arange(4, device="cuda")).all() and (ids[:, 4:] == -1).all()


def test_route_shapes_strides_and_empty():
    m = _mod()
    l = _rn(_gen(2), 2, 3, 24)
    w, ids = m.route(l, 2)
    assert w.shape == ids.shape == (2, 3, 2)
    w2, ids2 = m.route(l.transpose(0, 1).contiguous().transpose(0, 1), 2)
    assert torch.equal(w, w2) and torch.equal(ids, ids2)
    w, ids = m.route(l[:0].requires_grad_(), 2)
    assert w.shape == (0, 3, 2)
    plan = m.plan_experts(ids, 24)
    assert plan.offsets.tolist() == [0] * 25 and plan.order.numel() == 0


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _check_linear(T, k, E, D, N, gather, lost=0.0, seed=0, strided=False, skew=0.5):
    m, g = _mod(), _gen(seed)
    ids = _ids(T, k, E, g, lost, skew)
    plan = m.plan_experts(ids, E)
    R = T * k
    rows = T if gather else R
    x = _rn(g, rows, D + (24 if strided else 0)).to(BF)[:, :D]
    W = (0.1 * _rn(g, E, N, D)).to(BF)
    if strided:
        W = W.transpose(1, 2).contiguous().transpose(1, 2)
    dy = _rn(g, R, N + (8 if strided else 0)).to(BF)[:, :N]
    x.requires_grad_(), W.requires_grad_()
    y = m.expert_linear(x, W, plan, gather=gather)
    dx, dW = torch.autograd.grad(y, (x, W), dy)
    off, order = plan.offsets.tolist(), plan.order.long()
    xd, Wd, gd = x.detach().double(), W.detach().double(), dy.double()
    src = order // k if gather else torch.arange(R, device="cuda")
    want, mag = (torch.zeros(R, N, dtype=torch.float64, device="cuda") for _ in range(2))
    wdx, mdx = torch.zeros_like(xd), torch.zeros_like(xd)
    wdW, mdW = torch.zeros_like(Wd), torch.zeros_like(Wd)
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        xe, ge = xd[src[a:b]], gd[a:b]
        want[a:b], mag[a:b] = xe @ Wd[e].T, xe.abs() @ Wd[e].abs().T
        part, part_mag = ge @ Wd[e], ge.abs() @ Wd[e].abs()
        wdx.index_add_(0, src[a:b], part)
        mdx.index_add_(0, src[a:b], part_mag)
        wdW[e], mdW[e] = ge.T @ xe, ge.abs().T @ xe.abs()
    assert y.dtype == dx.dtype == dW.dtype == BF
    _close(y.detach(), want, mag, D, "y")
    _close(dW, wdW, mdW, max(b - a for a, b in zip(off, off[1:])), "dW")
    _close(dx, wdx, mdx, N + k, "dx")
    return y.detach(), dx, dW


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T,k,E,D,N", [
    (1, 1, 1, 8, 8), (1, 8, 64, 256, 128), (3, 2, 4, 64, 64), (17, 1, 3, 72, 40), (130, 2, 5, 200, 136), (300, 3, 7, 264, 520),
    (1000, 2, 8, 128, 384), (64, 1, 200, 96, 64), (2048, 2, 4, 768, 256), (515, 4, 16, 1024, 72)])
def test_linear(T, k, E, D, N, gather):
    _check_linear(T, k, E, D, N, gather)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T,k,E,D,N", [
    (4200, 1, 1, 136, 4104), (4360, 1, 1, 72, 4872), (4096, 2, 2, 200, 2312), (5000, 1, 1, 3912, 88), (9000, 2, 70, 520, 1032), (4700, 1, 1, 131, 4099)])
def test_linear_of_last_rounds_in_parts(T, k, E, D, N, gather):
    """A few tiles of 256 x 256 more than there are CUs: quarters and halves of them, some behind the last row and column."""
    _check_linear(T, k, E, D, N, gather)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("T,k,E,D,N", [(1, 1, 1, 1, 1), (5, 2, 3, 7, 9), (130, 3, 5, 201, 133), (260, 2, 37, 501, 333), (33, 1, 2, 63, 65), (40, 2, 6, 130, 258)])
def test_linear_odd(T, k, E, D, N, gather):
    _check_linear(T, k, E, D, N, gather, lost=0.2)


@pytest.mark.parametrize("gather", [False, True])
def test_linear_strided_and_skewed(gather):
    _check_linear(300, 2, 6, 128, 192, gather, strided=True)
    _check_linear(300, 2, 6, 100, 50, gather, strided=True, lost=0.3)
    _check_linear(700, 1, 32, 64, 128, gather, skew=30.0)       # nearly all to one expert


def test_linear_rows_behind_the_last_expert():
    """They are 0, and what x and the gradient hold there reaches nothing."""
    m, g = _mod(), _gen(5)
    T, k, E, D, N = 200, 2, 4, 64, 96
    ids = _ids(T, k, E, g)
    ids[120:] = -1
    plan = m.plan_experts(ids, E)
    used = int(plan.offsets[-1])
    assert used == 240
    x, W, dy = _rn(g, T * k, D).to(BF), _rn(g, E, N, D).to(BF), _rn(g, T * k, N).to(BF)
    x[used:], dy[used:] = torch.nan, torch.inf
    x.requires_grad_(), W.requires_grad_()
    y = m.expert_linear(x, W, plan)
    dx, dW = torch.autograd.grad(y, (x, W), dy)
    assert (y[used:] == 0).all() and (dx[used:] == 0).all()
    assert torch.isfinite(y).all() and torch.isfinite(dx).all() and torch.isfinite(dW).all()
    # gathered: tokens without a row
    t = _rn(g, T, D).to(BF)
    t[120:] = torch.nan
    t.requires_grad_()
    y = m.expert_linear(t, W, plan, gather=True)
    dt, dW = torch.autograd.grad(y, (t, W), dy)
    assert torch.isfinite(y).all() and torch.isfinite(dt).all() and torch.isfinite(dW).all() and (dt[120:] == 0).all()


@pytest.mark.parametrize("kept", [3052, 4355, 0])
def test_rows_behind_among_the_last_rounds_parts(kept):
    """Rows of no expert whose tiles are among those that go out in parts; results where a freed tensor of ones was."""
    m, g = _mod(), _gen(kept)
    T, D, N = 4360, 72, 4872
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    ids[torch.randperm(T, generator=g, device="cuda")[kept:]] = -1
    plan = m.plan_experts(ids, 1)
    order = plan.order[:kept].long()
    x, W = _rn(g, T, D).to(BF), _rn(g, 1, N, D).to(BF)
    x[ids[:, 0] < 0] = torch.nan
    del_me = torch.ones(T, N, dtype=BF, device="cuda")
    del del_me
    y = m.expert_linear(x, W, plan, gather=True)
    want = x[order].double() @ W[0].double().T
    _close(y[:kept], want, x[order].double().abs() @ W[0].double().abs().T, D, "y")
    assert (y[kept:] == 0).all()


def test_linear_stays_inside_its_expert():
    """NaN weights and rows of one expert reach no other one's results."""
    m, g = _mod(), _gen(6)
    T, k, E, D, N = 333, 1, 5, 72, 88
    ids = _ids(T, k, E, g)
    plan = m.plan_experts(ids, E)
    off = plan.offsets.tolist()
    x, W, dy = _rn(g, T, D).to(BF), _rn(g, E, N, D).to(BF), _rn(g, T, N).to(BF)
    W[2], x[off[2]:off[3]], dy[off[2]:off[3]] = torch.nan, torch.nan, torch.nan
    x.requires_grad_(), W.requires_grad_()
    y = m.expert_linear(x, W, plan)
    dx, dW = torch.autograd.grad(y, (x, W), dy)
    other = torch.ones(T, dtype=torch.bool, device="cuda")
    other[off[2]:off[3]] = False
    assert torch.isfinite(y[other]).all() and torch.isfinite(dx[other]).all()
    assert torch.isfinite(dW[[0, 1, 3, 4]]).all() and dW[2].isnan().all()


def test_linear_plans_out_of_range():
    """A plan with rows and offsets past its operands reads and writes nothing outside them."""
    m, g = _mod(), _gen(7)
    T, k, E, D, N = 50, 2, 3, 64, 64
    plan = m.plan_experts(_ids(T, k, E, g), E)
    x, W, w = _rn(g, T, D).to(BF), _rn(g, E, N, D).to(BF), torch.rand(T, k, device="cuda")
    want = m.expert_linear(x, W, plan, gather=True)
    bad = plan._replace(order=plan.order + 10 ** 6)
    assert (m.expert_linear(x, W, bad, gather=True) == 0).all()
    bad = plan._replace(offsets=torch.tensor([-5, 40, 10 ** 6, 7], device="cuda").int())
    y = m.expert_linear(x, W, bad, gather=True)
    assert torch.isfinite(y).all() and y.shape == want.shape
    bad = plan._replace(place=plan.place + 10 ** 6)
    assert (m.expert_combine(want, w, bad) == 0).all()


def test_linear_same_bits_every_call():
    a, b = (_check_linear(400, 2, 6, 136, 200, True, lost=0.1) for _ in range(2))
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_linear_only_what_is_asked_for():
    m, g = _mod(), _gen(8)
    plan = m.plan_experts(_ids(40, 2, 4, g), 4)
    x, W = _rn(g, 40, 64).to(BF), _rn(g, 4, 32, 64).to(BF)
    kept = []
    hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(tuple(t.shape)) or t, lambda t: t)
    with hooks:
        y = m.expert_linear(x.clone().requires_grad_(), W, plan, gather=True)
    assert tuple(W.shape) in kept and tuple(x.shape) not in kept
    y.sum().backward()
    kept.clear()
    Wg = W.clone().requires_grad_()
    with hooks:
        y = m.expert_linear(x, Wg, plan, gather=True)
    assert tuple(W.shape) not in kept and tuple(x.shape) in kept
    y.sum().backward()
    assert Wg.grad.shape == W.shape


# ---------------------------------------------------------------------------
# the weighted sum
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,E,D,lost", [(1, 1, 1, 1, 0.0), (1, 8, 64, 512, 0.0), (37, 3, 5, 201, 0.2), (300, 2, 8, 768, 0.0), (64, 64, 64, 40, 0.5),
                                          (130, 4, 9, 4104, 0.1), (20, 2, 4, 2049, 1.0)])
def test_combine(T, k, E, D, lost):
    m, g = _mod(), _gen(T + D)
    plan = m.plan_experts(_ids(T, k, E, g, lost), E)
    y = _rn(g, T * k, D + 5).to(BF)[:, :D].requires_grad_()
    w = _rn(g, T, k).requires_grad_()
    go = _rn(g, T, D).to(BF)
    out = m.expert_combine(y, w, plan)
    dy, dw = torch.autograd.grad(out, (y, w), go)
    place = plan.place.long()
    there = (place >= 0)[..., None]
    terms = torch.where(there, w.detach().double()[..., None] * y.detach().double()[place.clamp(min=0)], 0.0)
    _close(out.detach(), terms.sum(1), terms.abs().sum(1), k, "out")
    dots = torch.where(there, y.detach().double()[place.clamp(min=0)] * go.double()[:, None], 0.0)
    _close(dw, dots.sum(-1), dots.abs().sum(-1), D, "dw")
    want = torch.zeros(T * k, D, dtype=torch.float64, device="cuda")
    want[place[there[..., 0]]] = (w.detach().double()[..., None] * go.double()[:, None])[there[..., 0]]
    _close(dy, want, want.abs(), 1, "dy")
    # one gradient without the other
    a, = torch.autograd.grad(m.expert_combine(y, w.detach(), plan), y, go)
    b, = torch.autograd.grad(m.expert_combine(y.detach(), w, plan), w, go)
    assert torch.equal(a, dy) and torch.equal(b, dw)


def test_a_block_of_experts():
    """Routing, both products, the sum: as they are used, forward and backward, twice the same; token shapes kept."""
    m, g = _mod(), _gen(9)
    B, S, D, H, E, k = 3, 50, 128, 96, 8, 2
    x = _rn(g, B, S, D).to(BF).requires_grad_()
    Wr = (0.1 * _rn(g, E, D)).to(BF).requires_grad_()
    W1, W2 = ((0.1 * _rn(g, *s)).to(BF).requires_grad_() for s in ((E, H, D), (E, D, H)))
    go = _rn(g, B, S, D).to(BF)

    def step():
        w, ids = m.route(x @ Wr.T, k)
        plan = m.plan_experts(ids, E)
        h = torch.relu(m.expert_linear(x, W1, plan, gather=True))
        out = m.expert_combine(m.expert_linear(h, W2, plan), w, plan)
        return out, torch.autograd.grad(out, (x, Wr, W1, W2), go)
    out, grads = step()
    out2, grads2 = step()
    assert out.shape == (B, S, D) and torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    # dense: every expert on every token, weighted
    xd, W1d, W2d, Wrd = (t.detach().double().requires_grad_() for t in (x, W1, W2, Wr))
    logits = (x @ Wr.T).detach().double() + (xd @ Wrd.T - (xd @ Wrd.T).detach())
    ids = m.route((x @ Wr.T).detach(), k)[1].long()
    s = torch.softmax(logits, -1).gather(-1, ids)
    w = torch.zeros(B, S, E, dtype=torch.float64, device="cuda").scatter(-1, ids, s / s.sum(-1, keepdim=True))
    y = torch.stack([torch.relu(xd @ W1d[e].T) @ W2d[e].T for e in range(E)], -1)
    ref = (y * w[:, :, None]).sum(-1)
    want = torch.autograd.grad(ref, (xd, Wrd, W1d, W2d), go.double())
    # bf16 results in between: three on the way, five back, each 2^-9 rms of its size
    for name, a, b in zip(("out", "x", "Wr", "W1", "W2"), (out, *grads), (ref, *want)):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel < 8 * 2.0 ** -8, (name, rel)
