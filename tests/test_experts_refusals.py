"""What the experts' and dropout's Python calls refuse: their arguments on the CPU, their operands on the GPU, forward-mode
tangents and function transforms."""
import pytest
import torch
from torch.autograd import forward_ad

from bitsparse_amd.dropout import Dropout, dropout
from bitsparse_amd.experts import ExpertPlan, ExpertsRelu, expert_combine, expert_linear, plan_experts, route
from bitsparse_amd.residual import block_join

BF, I32 = torch.bfloat16, torch.int32


def test_arguments():
    x = torch.ones(4, 8)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="drop.p"):
            dropout(x, Dropout(p, 0))
    for kw in (dict(seed=-1), dict(seed=2 ** 64), dict(seed=0, offset=-1), dict(seed=0, offset=2 ** 64)):
        with pytest.raises(ValueError, match="2\\^64"):
            dropout(x, Dropout(0.5, **kw))
    with pytest.raises(ValueError, match="offset"):
        dropout(x, Dropout(0.5, torch.zeros(2, dtype=torch.int64), 3))
    for drop in (0.5, (0.5, 1), None):
        with pytest.raises(TypeError, match="Dropout"):
            dropout(x, drop)
    with pytest.raises(TypeError, match="Dropout"):
        block_join(x, x, drop=0.1)
    with pytest.raises(ValueError, match="score"):
        route(x, 2, score="relu")


def test_cpu_tensors():
    x, plan = torch.ones(4, 8, dtype=BF), ExpertPlan(torch.zeros(3, dtype=I32), torch.zeros(8, dtype=I32), torch.zeros(4, 2, dtype=I32))
    W = torch.ones(2, 8, 8, dtype=BF)
    for call in (lambda: dropout(x, Dropout(0.5, 0)), lambda: route(x, 2), lambda: plan_experts(torch.zeros(4, 2, dtype=I32), 2),
                 lambda: expert_linear(x, W, plan, gather=True), lambda: expert_combine(torch.ones(8, 8, dtype=BF), torch.ones(4, 2), plan),
                 lambda: ExpertsRelu.apply(x, W, W, torch.ones(4, 2), plan), lambda: block_join(x, x, drop=Dropout(0.5, 0))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.gpu
def test_operands():
    dev = "cuda"
    l = torch.randn(6, 16, device=dev)
    bad = [
        (TypeError, "logits", lambda: route(l.half(), 2)), (ValueError, "top_k", lambda: route(l, 0)), (ValueError, "top_k", lambda: route(l, 17)),
        (ValueError, "groups", lambda: route(l, 2, groups=3)), (ValueError, "top_groups", lambda: route(l, 2, groups=4, top_groups=5)),
        (ValueError, "more than", lambda: route(l, 5, groups=4, top_groups=1)), (ValueError, "group_best", lambda: route(l, 2, groups=4, top_groups=2, group_best=3)),
        (TypeError, "bias", lambda: route(l, 2, bias=torch.zeros(16, device=dev).bfloat16())), (ValueError, "bias", lambda: route(l, 2, bias=torch.zeros(15, device=dev))),
        (RuntimeError, "bias", lambda: route(l, 2, bias=torch.zeros(16))), (ValueError, "experts", lambda: route(torch.randn(3, 2000, device=dev), 2)),
        (ValueError, "logits", lambda: route(torch.zeros(3, 0, device=dev), 1)),
        (TypeError, "int32", lambda: plan_experts(torch.zeros(4, 2, device=dev, dtype=torch.int64), 4)),
        (ValueError, "n_experts", lambda: plan_experts(torch.zeros(4, 2, device=dev, dtype=I32), 0)),
        (ValueError, "n_experts", lambda: plan_experts(torch.zeros(4, 2, device=dev, dtype=I32), 1025))]
    w, ids = route(l, 2)
    plan = plan_experts(ids, 16)
    x, rows, W = torch.randn(6, 32, device=dev).to(BF), torch.randn(12, 32, device=dev).to(BF), torch.randn(16, 24, 32, device=dev).to(BF)
    bad += [
        (TypeError, "x must", lambda: expert_linear(x.float(), W, plan, gather=True)), (TypeError, "W must", lambda: expert_linear(rows, W.float(), plan)),
        (ValueError, "12 rows", lambda: expert_linear(x, W, plan)), (ValueError, "6 tokens", lambda: expert_linear(rows, W, plan, gather=True)),
        (ValueError, "W: expected", lambda: expert_linear(rows, W[:15], plan)), (ValueError, "32 columns", lambda: expert_linear(rows, W[..., :31], plan)),
        (ValueError, "experts, out, in", lambda: expert_linear(rows, W[0], plan)), (RuntimeError, "GPU", lambda: expert_linear(rows.cpu(), W, plan)),
        (TypeError, "plan.order", lambda: expert_linear(rows, W, plan._replace(order=plan.order.long()))),
        (ValueError, "plan.order", lambda: expert_linear(rows, W, plan._replace(order=plan.order[:-1]))),
        (ValueError, "plan.offsets", lambda: expert_linear(rows, W, plan._replace(offsets=plan.offsets[:1]))),
        (ValueError, "plan.place", lambda: expert_linear(rows, W, plan._replace(place=plan.place.view(1, 12).expand(1, 12).repeat(1, 6)))),
        (RuntimeError, "GPU", lambda: expert_linear(rows, W, plan._replace(place=plan.place.cpu()))),
        (TypeError, "y must", lambda: expert_combine(rows.float(), w, plan)), (TypeError, "weights", lambda: expert_combine(rows, w.to(BF), plan)),
        (ValueError, "weights", lambda: expert_combine(rows, w[:5], plan)), (ValueError, "12 rows", lambda: expert_combine(rows[:11], w, plan)),
        (ValueError, "W: expected", lambda: ExpertsRelu.apply(x, W, W, w, plan)),
        (TypeError, "x must", lambda: dropout(x.half(), Dropout(0.5, 0))),
        (TypeError, "int64", lambda: dropout(x, Dropout(0.5, torch.zeros(2, device=dev, dtype=I32)))),
        (ValueError, "seed", lambda: dropout(x, Dropout(0.5, torch.zeros(3, device=dev, dtype=torch.int64)))),
        (RuntimeError, "GPU", lambda: dropout(x, Dropout(0.5, torch.zeros(2, dtype=torch.int64))))]
    for i, (error, word, call) in enumerate(bad):
        with pytest.raises(error, match=word):
            call()
            pytest.fail(f"{i}: {word}")


@pytest.mark.gpu
def test_gradients_are_checked():
    dev = "cuda"
    l = torch.randn(6, 16, device=dev).requires_grad_()
    w, ids = route(l, 2)
    plan = plan_experts(ids, 16)
    rows, W = torch.randn(12, 32, device=dev).to(BF).requires_grad_(), torch.randn(16, 24, 32, device=dev).to(BF).requires_grad_()
    y = expert_linear(rows, W, plan)
    out = expert_combine(y, w, plan)
    for t, inputs in ((w, [l]), (y, [rows, W]), (out, [y, w])):
        with pytest.raises(NotImplementedError, match="second derivative"):
            torch.autograd.grad(t, inputs, torch.ones_like(t), create_graph=True)
    # what hooks hand back instead of the saved tensors
    swap = {"W": lambda t: t[:, :, :16] if t.shape == W.shape else t, "x": lambda t: t.float() if t.shape == rows.shape else t,
            "plan.order": lambda t: t[:-1] if t.shape == plan.order.shape else t}
    for name, f in swap.items():
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, f):
            y = expert_linear(rows, W, plan)
        with pytest.raises((RuntimeError, ValueError, TypeError), match=name):
            torch.autograd.grad(y, [rows, W], torch.ones_like(y))


@pytest.mark.gpu
def test_in_place_changes_are_seen():
    """An operand that changed between forward and backward is an error, not a wrong gradient."""
    dev = "cuda"
    w, ids = route(torch.randn(6, 16, device=dev), 2)
    plan = plan_experts(ids, 16)
    rows, W = torch.randn(12, 32, device=dev).to(BF).requires_grad_(), torch.randn(16, 24, 32, device=dev).to(BF)
    y = expert_linear(rows, W, plan)
    W.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, rows, torch.ones_like(y))


def _calls():
    l = torch.randn(6, 16, device="cuda")
    w, ids = route(l, 2)
    plan = plan_experts(ids, 16)
    x, rows, W = torch.randn(6, 32, device="cuda").to(BF), torch.randn(12, 32, device="cuda").to(BF), torch.randn(16, 32, 32, device="cuda").to(BF)
    yield "logits", l, lambda d: route(d, 2)
    yield "x gathered", x, lambda d: expert_linear(d, W, plan, gather=True)
    yield "x", rows, lambda d: expert_linear(d, W, plan)
    yield "W", W, lambda d: expert_linear(rows, d, plan)
    yield "y", rows, lambda d: expert_combine(d, w, plan)
    yield "weights", w, lambda d: expert_combine(rows, d, plan)
    yield "dropped", x, lambda d: dropout(d, Dropout(0.5, 0))
    yield "joined", x, lambda d: block_join(x, d, drop=Dropout(0.5, 0))
    yield "x of a block", x, lambda d: ExpertsRelu.apply(d, W, W, w, plan)
    yield "W2 of a block", W, lambda d: ExpertsRelu.apply(x, W, d, w, plan)


@pytest.mark.gpu
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents(requires_grad):
    for name, t, call in _calls():
        t = t.detach().clone().requires_grad_(requires_grad)
        with forward_ad.dual_level():
            with pytest.raises((NotImplementedError, RuntimeError), match="forward"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
                pytest.fail(name)
        call(t)


@pytest.mark.gpu
def test_transforms():
    for name, t, call in _calls():
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.vmap(lambda d: call(d)[0])(t[None])
            pytest.fail(name)
