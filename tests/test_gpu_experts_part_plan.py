"""Plans of some of the experts: offsets[e0:e1 + 1] of a plan of all with W[e0:e1], whose rows begin behind row 0 and end before
the last.  The rows outside belong to no expert: results and gradients are 0 there, whatever the memory held before.

Bars as in tests/test_gpu_experts.py and tests/test_gpu_experts_block.py.
"""
import pytest
import torch
from test_gpu_experts import BF, _close, _gen, _ids, _rn

pytestmark = pytest.mark.gpu


def _dirty(*sizes):
    """Leaves blocks of these many bytes, all NaN, for the allocator to hand out next."""
    torch.cuda.synchronize()
    held = [torch.full(((n + 3) // 4,), torch.nan, device="cuda") for n in sizes for _ in range(3)]
    del held


def _part(ids, E, e0, e1, own):
    """The plan of experts e0 up to e1; own: pairs of the other experts have no row in it."""
    from bitsparse_amd.experts import ExpertPlan, plan_experts
    plan = plan_experts(ids, E)
    first, end = int(plan.offsets[e0]), int(plan.offsets[e1])
    order, place = plan.order, plan.place
    if own:
        r = torch.arange(order.numel(), device="cuda")
        order = torch.where((r >= first) & (r < end), order, -1)
        place = torch.where((place >= first) & (place < end), place, -1)
    return plan, ExpertPlan(plan.offsets[e0:e1 + 1], order, place), first, end


# rows one or two an expert; tiles of every size; odd sizes; an expert without rows before and behind all the rows
PARTS = [(4, 2, 64, 20, 60, 256, 128), (1, 1, 3, 2, 3, 64, 64), (130, 2, 5, 1, 4, 72, 136), (130, 3, 5, 1, 3, 201, 133), (700, 2, 130, 70, 129, 128, 192),
         (4096, 4, 4, 1, 3, 256, 512), (8192, 2, 8, 3, 6, 384, 1024), (4700, 1, 3, 1, 3, 72, 4872), (50, 1, 3, 1, 2, 64, 64)]


@pytest.mark.parametrize("T,k,E,e0,e1,D,N", PARTS)
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_linear(T, k, E, e0, e1, D, N, own, gather):
    from bitsparse_amd.experts import expert_linear
    g = _gen(T + D)
    ids = _ids(T, k, E, g, lost=0.1)
    if T == 50:
        ids[:30], ids[30:] = 0, 2                       # none of the one expert's
    full, plan, first, end = _part(ids, E, e0, e1, own)
    R = T * k
    x, W, dy = _rn(g, T if gather else R, D).to(BF), (0.1 * _rn(g, e1 - e0, N, D)).to(BF), _rn(g, R, N).to(BF)
    x.requires_grad_(), W.requires_grad_()
    _dirty(2 * R * N, 4 * R * D, 2 * R * D)
    y = expert_linear(x, W, plan, gather=gather)
    dx, dW = torch.autograd.grad(y, (x, W), dy)
    off = full.offsets.tolist()
    src = full.order.long() // k if gather else torch.arange(R, device="cuda")
    xd, Wd, gd = x.detach().double(), W.detach().double(), dy.double()
    want, mag = (torch.zeros(R, N, dtype=torch.float64, device="cuda") for _ in range(2))
    wdx, mdx, wdW, mdW = torch.zeros_like(xd), torch.zeros_like(xd), torch.zeros_like(Wd), torch.zeros_like(Wd)
    for e in range(e0, e1):
        a, b = off[e], off[e + 1]
        xe, ge, We = xd[src[a:b]], gd[a:b], Wd[e - e0]
        want[a:b], mag[a:b] = xe @ We.T, xe.abs() @ We.abs().T
        wdx.index_add_(0, src[a:b], ge @ We)
        mdx.index_add_(0, src[a:b], ge.abs() @ We.abs())
        wdW[e - e0], mdW[e - e0] = ge.T @ xe, ge.abs().T @ xe.abs()
    assert (y[:first] == 0).all() and (y[end:] == 0).all()
    _close(y.detach(), want, mag, D, "y")
    _close(dx, wdx, mdx, N + k, "dx")
    _close(dW, wdW, mdW, R, "dW")


@pytest.mark.parametrize("offsets", [[40, 40], [0, 0], [40, 40, 40], [17, 17, 40]])
def test_offsets_at_an_end(offsets):
    """All the rows before the first expert's, or behind the last one's."""
    from bitsparse_amd.experts import ExpertPlan, expert_linear
    g = _gen(1)
    at = torch.arange(40, device="cuda", dtype=torch.int32)
    plan = ExpertPlan(torch.tensor(offsets, device="cuda", dtype=torch.int32), at, at[:, None].clone())
    x, W = _rn(g, 40, 64).to(BF), _rn(g, len(offsets) - 1, 32, 64).to(BF).requires_grad_()
    x.requires_grad_()
    _dirty(40 * 64 * 2, 40 * 32 * 2)
    y = expert_linear(x, W, plan)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    first, end = offsets[0], offsets[-1]
    assert (y[:first] == 0).all() and (y[end:] == 0).all() and (dx[:first] == 0).all() and (dx[end:] == 0).all()
    want = x.detach()[first:end].double() @ W.detach()[-1].double().T
    _close(y.detach()[first:end], want, x.detach()[first:end].double().abs() @ W.detach()[-1].double().abs().T, 64, "y")


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("T,k,E,e0,e1,D,H,O", [(40, 2, 4, 1, 3, 72, 136, 40), (200, 3, 8, 2, 7, 128, 256, 128), (33, 4, 16, 15, 16, 65, 131, 67), (2, 2, 32, 8, 24, 64, 64, 64)])
def test_block(T, k, E, e0, e1, D, H, O, square, own):
    """A block of some of the experts is their share of the sum: gradients reach their weights and tokens, and no others."""
    from bitsparse_amd.experts import ExpertsRelu, ExpertsRelu2
    from test_gpu_experts_block import _inputs, _near, _reference
    layer = ExpertsRelu2 if square else ExpertsRelu
    t, ids, _, go = _inputs(T, E, k, D, H, O, 0.1)
    _, plan, _, _ = _part(ids, E, e0, e1, own)
    t["W1"], t["W2"] = t["W1"][e0:e1].clone(), t["W2"][e0:e1].clone()
    mine = torch.where((ids >= e0) & (ids < e1), ids - e0, -1)
    for a in t.values():
        a.requires_grad_()
    R = T * k
    _dirty(2 * R * H, 2 * R * O, 4 * R * D)
    out = layer.apply(*t.values(), plan)
    grads = dict(zip(t, torch.autograd.grad(out, list(t.values()), go)))
    want, want_grads = _reference(t, mine, go, square)
    _near(out.detach(), want, "out")
    for n in t:
        assert torch.isfinite(grads[n]).all(), n
        if want_grads[n].norm() > 0:
            _near(grads[n], want_grads[n], n)
    assert (grads["w"][mine < 0] == 0).all()
    with torch.no_grad():
        assert torch.equal(layer.apply(*t.values(), plan), out)


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("T,k,E,e0,e1,D", [(1, 1, 3, 2, 3, 8), (40, 2, 4, 1, 3, 72), (130, 3, 5, 1, 3, 201), (300, 4, 8, 3, 6, 4104), (50, 1, 3, 1, 2, 64),
                                           (2, 64, 64, 10, 40, 33)])
def test_combine(T, k, E, e0, e1, D, own):
    """Whatever y holds in rows of no expert is in no sum; the gradients there are 0, in every call the same."""
    from bitsparse_amd.experts import expert_combine
    g = _gen(T + D)
    ids = _ids(T, k, E, g, lost=0.1)
    if T == 50:
        ids[:30], ids[30:] = 0, 2
    _, plan, first, end = _part(ids, E, e0, e1, own)
    R = T * k
    y, w, go = _rn(g, R, D).to(BF), _rn(g, T, k).requires_grad_(), _rn(g, T, D).to(BF)
    y[:first], y[end:] = torch.nan, torch.inf
    y.requires_grad_()
    mine = (ids >= e0) & (ids < e1)
    at = plan.place.long().clamp(min=0)
    rows = torch.where(mine[..., None], y.detach().double()[at], 0.0)
    terms, dots = w.detach().double()[..., None] * rows, rows * go.double()[:, None]
    want = torch.zeros(R, D, dtype=torch.float64, device="cuda")
    want[at[mine]] = (w.detach().double()[..., None] * go.double()[:, None])[mine]
    for _ in range(3):
        _dirty(2 * R * D, 4 * R)
        out = expert_combine(y, w, plan)
        dy, dw = torch.autograd.grad(out, (y, w), go)
        _close(out.detach(), terms.sum(1), terms.abs().sum(1), k, "out")
        _close(dw, dots.sum(-1), dots.abs().sum(-1), D, "dw")
        _close(dy, want, want.abs(), 1, "dy")
        assert (dy[:first] == 0).all() and (dy[end:] == 0).all() and (dw[~mine] == 0).all()
        _dirty(2 * R * D)
        alone, = torch.autograd.grad(expert_combine(y, w.detach(), plan), y, go)
        assert torch.equal(alone, dy)
