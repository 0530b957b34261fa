"""Blocks of experts whose activation is saved compressed (ExpertsRelu, ExpertsRelu2) against the same in 64 bits.

Bars.  Results that follow one another are each rounded to bf16 (a relative
error of 2^-9 in the mean, independent of one another): on the way to the
output z, the activation (twice for ReLU^2, which doubles z's error too), y and
the sum; to a gradient those of the activation and the gradients of y, of the
activation and of z besides the result.  At most ten such, each of 2^-9 / sqrt(3)
of the 2-norm and doubled at most: under 10 * 2^-9 in the sum of squares' root.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
BAR = 10 * 2.0 ** -9


def _inputs(T, E, k, D, H, O, lost, seed=0, shape=None):
    from bitsparse_amd.experts import plan_experts, route
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    logits = rn(T, E)
    if lost:
        logits[torch.rand(T, generator=g, device="cuda") < lost] = -torch.inf
    w, ids = route(logits, k, score="sigmoid")
    t = {"x": rn(T, D).to(BF), "W1": (rn(E, H, D) * D ** -0.5).to(BF), "W2": (rn(E, O, H) * H ** -0.5).to(BF), "w": w}
    if shape:
        t["x"], t["w"], ids = t["x"].view(*shape, D), w.view(*shape, k), ids.view(*shape, k)
    plan = plan_experts(ids, E)
    return t, ids, plan, rn(*(shape or (T,)), O).to(BF)


def _reference(t, ids, go, square):
    v = {n: a.detach().double().requires_grad_() for n, a in t.items()}
    x, w, e = v["x"].reshape(-1, v["x"].shape[-1]), v["w"].reshape(-1, v["w"].shape[-1]), ids.reshape(-1, ids.shape[-1]).long()
    E = v["W1"].shape[0]
    dense = torch.zeros(x.shape[0], E + 1, dtype=torch.float64, device="cuda").scatter(1, torch.where(e < 0, E, e), w)[:, :E]
    out = 0
    for i in range(E):
        r = torch.relu(x @ v["W1"][i].T)
        out = out + dense[:, i:i + 1] * ((r * r if square else r) @ v["W2"][i].T)
    grads = torch.autograd.grad(out, list(v.values()), go.double().reshape(out.shape))
    return out.detach(), dict(zip(v, grads))


def _near(got, want, name):
    want = want.reshape(got.shape)
    assert torch.isfinite(got).all(), name
    err = (got.double() - want).norm() / want.norm().clamp(min=1e-30)
    assert err < BAR, (name, err.item())


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("T,E,k,D,H,O,lost", [(1, 1, 1, 64, 64, 64, 0.0), (40, 4, 2, 72, 136, 40, 0.0), (200, 8, 3, 128, 256, 128, 0.3), (33, 16, 4, 65, 131, 67, 0.2),
                                              (512, 8, 2, 256, 512, 256, 0.0)])
@pytest.mark.parametrize("storage", ["buffer", "packed", "none"])
def test_block(square, T, E, k, D, H, O, lost, storage):
    from bitsparse_amd.bitsparse import TensorBuffer
    from bitsparse_amd.experts import ExpertsRelu, ExpertsRelu2
    layer = ExpertsRelu2 if square else ExpertsRelu
    t, ids, plan, go = _inputs(T, E, k, D, H, O, lost)
    for a in t.values():
        a.requires_grad_()
    packed = storage == "packed"
    buf = None if storage == "none" else TensorBuffer(2 * T * k * H + 64, device="cuda", pack_sbit=packed)
    out = layer.apply(t["x"], t["W1"], t["W2"], t["w"], plan, sparse_data=buf, pack_sbit=packed)
    grads = dict(zip(t, torch.autograd.grad(out, list(t.values()), go)))
    want, want_grads = _reference(t, ids, go, square)
    _near(out.detach(), want, "out")
    for n in t:
        assert grads[n].shape == t[n].shape and grads[n].dtype == t[n].dtype
        if want_grads[n].norm() > 0:
            _near(grads[n], want_grads[n], n)
    assert (grads["w"][ids < 0] == 0).all()
    if buf is not None:
        assert not buf.overflowed()
    # without gradients the same values
    with torch.no_grad():
        plain = layer.apply(t["x"], t["W1"], t["W2"], t["w"], plan)
    assert torch.equal(plain, out)


def test_tokens_keep_their_shape():
    from bitsparse_amd.experts import ExpertsRelu2
    t, ids, plan, go = _inputs(24, 4, 2, 64, 96, 32, 0.0, shape=(2, 3, 4))
    for a in t.values():
        a.requires_grad_()
    out = ExpertsRelu2.apply(*t.values(), plan)
    assert out.shape == (2, 3, 4, 32)
    want, want_grads = _reference(t, ids, go, True)
    _near(out.detach(), want, "out")
    for n, g in zip(t, torch.autograd.grad(out, list(t.values()), go)):
        assert g.shape == t[n].shape
        _near(g, want_grads[n], n)


def test_only_what_is_asked_for():
    """Each gradient alone is the one that all together give; the weights' alone; none at all."""
    from bitsparse_amd.experts import ExpertsRelu2
    t, ids, plan, go = _inputs(60, 4, 2, 64, 128, 48, 0.2)
    for a in t.values():
        a.requires_grad_()
    full = torch.autograd.grad(ExpertsRelu2.apply(*t.values(), plan), list(t.values()), go)
    for i, n in enumerate(t):
        one, = torch.autograd.grad(ExpertsRelu2.apply(*t.values(), plan), t[n], go)
        assert torch.equal(one, full[i])
        alone = {m: (a if m == n else a.detach()) for m, a in t.items()}
        one, = torch.autograd.grad(ExpertsRelu2.apply(*alone.values(), plan), t[n], go)
        assert torch.equal(one, full[i])
    out = ExpertsRelu2.apply(*(a.detach() for a in t.values()), plan)
    assert not out.requires_grad


def test_saves_its_activation_compressed():
    """What stays between forward and backward: the inputs, the plan and the compressed activation, no [rows, d_out]."""
    from bitsparse_amd.bitsparse import TensorBuffer
    from bitsparse_amd.experts import ExpertsRelu
    t, ids, plan, go = _inputs(4096, 4, 2, 256, 512, 512, 0.0)
    for a in t.values():
        a.requires_grad_()
    rows, H, O = 8192, 512, 512
    buf = TensorBuffer(rows * H, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = ExpertsRelu.apply(*t.values(), plan, sparse_data=buf)
    kept = torch.cuda.memory_allocated() - before - out.numel() * 2
    # bitmask, prefix and small change; the values are in the buffer
    assert kept <= rows * H // 8 + rows * H // 1024 + (1 << 20)


def test_goes_backward_once_and_not_twice():
    from bitsparse_amd.experts import ExpertsRelu
    t, ids, plan, go = _inputs(20, 2, 1, 32, 64, 32, 0.0)
    for a in t.values():
        a.requires_grad_()
    out = ExpertsRelu.apply(*t.values(), plan)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(out, list(t.values()), go, create_graph=True)
    out = ExpertsRelu.apply(*t.values(), plan)
    torch.autograd.grad(out, list(t.values()), go, retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out, list(t.values()), go)


def test_no_tokens():
    from bitsparse_amd.experts import ExpertsRelu2, plan_experts
    plan = plan_experts(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 3)
    x, W1, W2 = torch.zeros(0, 16, device="cuda").to(BF), torch.randn(3, 24, 16, device="cuda").to(BF), torch.randn(3, 8, 24, device="cuda").to(BF)
    w = torch.zeros(0, 2, device="cuda")
    for a in (x, W1, W2, w):
        a.requires_grad_()
    with torch.no_grad():
        assert ExpertsRelu2.apply(x, W1, W2, w, plan).shape == (0, 8)
    out = ExpertsRelu2.apply(x, W1, W2, w, plan)
    grads = torch.autograd.grad(out, (x, W1, W2, w), torch.zeros_like(out))
    assert out.shape == (0, 8) and all((g == 0).all() for g in grads)


def test_a_model_of_them():
    """Routing, a block of experts, dropout and the residual step with the next norm, forward and backward: all as one
    training step would use them, twice the same; gradients reach every parameter."""
    from bitsparse_amd.bitsparse import TensorBuffer
    from bitsparse_amd.dropout import Dropout
    from bitsparse_amd.experts import ExpertsRelu2, plan_experts, route
    from bitsparse_amd.residual import RowNorm, block_join, block_norm
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    B, S, D, H, E, k, L = 2, 65, 128, 256, 8, 2, 3
    P = [{"norm": torch.ones(D, device="cuda").to(BF), "Wr": (rn(E, D) * D ** -0.5).to(BF), "W1": (rn(E, H, D) * D ** -0.5).to(BF),
          "W2": (rn(E, D, H) * H ** -0.5).to(BF)} for _ in range(L)]
    last = torch.ones(D, device="cuda").to(BF)
    params = [p for d in P for p in d.values()] + [last]
    for p in params:
        p.requires_grad_()
    x0, go = rn(B, S, D), rn(B, S, D).to(BF)

    def step():
        buf = TensorBuffer(L * B * S * k * H + 64 * L, device="cuda")
        x, h = x0, block_norm(x0, RowNorm(P[0]["norm"]), dtype=BF)
        for i, p in enumerate(P):
            w, ids = route((h @ p["Wr"].T).float(), k, score="softmax")
            y = ExpertsRelu2.apply(h, p["W1"], p["W2"], w, plan_experts(ids, E), sparse_data=buf)
            x, h = block_join(x, y, drop=Dropout(0.1, 42, i), pre=RowNorm(P[i + 1]["norm"] if i + 1 < L else last))
        return (h, *torch.autograd.grad(h, params, go))
    a, b = step(), step()
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    assert all(torch.isfinite(t).all() for t in a) and all((t != 0).any() for t in a)
