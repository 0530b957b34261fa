"""What the step between two blocks keeps for its backward: what some gradient is formed of and nothing else, so that
the rest may be freed or changed in place."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
NAMES = ("x", "y", "w_post", "b_post", "gate", "scale", "w_pre", "b_pre")
T, D = 37, 200


def _mod():
    from bitsparse_amd import residual
    return residual


def _operands(gate="channel", dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(5)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    shape = {"one": (1,), "channel": (D,), "row": (T, 1), "element": (T, D)}[gate]
    t = {"x": rn(T, D), "y": rn(T, D), "w_post": 1 + rn(D), "b_post": rn(D), "gate": rn(*shape), "scale": rn(D), "w_pre": 1 + rn(D), "b_pre": rn(D)}
    return t, rn(T, D), rn(T, D)


def _call(t, post="rms", pre="rms"):
    R = _mod()
    out = R.block_join(t["x"], t["y"], post=R.RowNorm(t["w_post"], t["b_post"], post) if post else None, gate=t["gate"],
                       scale=t["scale"], pre=R.RowNorm(t["w_pre"], t["b_pre"], pre) if pre else None)
    return out if pre else (out,)


def _learn(t, names):
    return {k: v.clone().requires_grad_(k in names) for k, v in t.items()}


def _saved(t, post, pre, **kw):
    """addresses of what is kept, and the results"""
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v.data_ptr()) or v, lambda v: v):
        out = _call(t, post, pre, **kw)
    return set(kept), out


@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", None), (None, "rms"), (None, None)])
@pytest.mark.parametrize("learn", [("x",), ("y",), ("x", "y"), ("scale",), ("gate",), ("w_post",), ("b_post", "x"), ("w_pre", "b_pre"), NAMES])
def test_what_is_kept(post, pre, learn):
    learn = [k for k in learn if (post or not k.endswith("post")) and (pre or not k.endswith("pre"))]
    if not learn:
        return
    t = _learn(_operands()[0], learn)
    kept, out = _saved(t, post, pre)
    assert (t["x"].data_ptr() in kept) == ("scale" in learn)
    assert (t["y"].data_ptr() in kept) == ("gate" in learn or bool(post and {"y", "w_post"} & set(learn)))
    assert (out[0].data_ptr() in kept) == (pre is not None)
    assert t["b_pre"].data_ptr() not in kept
    assert (t["b_post"].data_ptr() in kept) == (post is not None and "gate" in learn)


def test_norm_alone_keeps_its_input():
    R = _mod()
    x = torch.randn(5, 64, device="cuda", requires_grad=True)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v.data_ptr()) or v, lambda v: v):
        R.block_norm(x, R.RowNorm())
    assert x.data_ptr() in kept


@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms"), (None, "layer"), ("rms", None), (None, None)])
@pytest.mark.parametrize("gate", ["one", "channel", "row", "element"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_that_learns(post, pre, gate, dtype):
    """The gradients of one or two operands that learn alone are those of all of them learning."""
    t, g_x, g_h = _operands(gate, dtype)
    names = [k for k in NAMES if (post or not k.endswith("post")) and (pre or not k.endswith("pre"))]
    seeds = (g_x, g_h)[:2 if pre else 1]
    full = _learn(t, names)
    want = dict(zip(names, torch.autograd.grad(_call(full, post, pre), [full[k] for k in names], seeds)))
    for some in [(k,) for k in names] + list(itertools.combinations(names, 2)):
        one = _learn(t, some)
        out = _call(one, post, pre)
        if not any(o.requires_grad for o in out):
            continue
        for k, g in zip(some, torch.autograd.grad(out, [one[k] for k in some], seeds, allow_unused=True)):
            # (two forms of the kernel: each within half a unit and 2^-19 of its terms, here at most eight times the largest)
            unit = 2.0 ** -7 if dtype == BF else 2.0 ** -23
            assert ((g - want[k]).abs() <= unit * want[k].abs() + 2.0 ** -15 * want[k].abs().max()).all(), (some, k)


def test_changed_in_place():
    """What no gradient is formed of may be overwritten before the backward; what one is formed of may not."""
    t, g_x, g_h = _operands()

    def grads(change, post, pre, seeds, names):
        c = _learn(t, names)
        out = _call(c, post, pre)
        change(c, out)
        return torch.autograd.grad(out, [c[k] for k in names], seeds)
    for change, post, pre, seeds, names in (
            (lambda c, out: (c["x"].zero_(), c["b_pre"].zero_(), c["b_post"].zero_()), "rms", "rms", (g_x, g_h), ("y", "w_pre")),
            (lambda c, out: (c["x"].zero_(), out[0].detach().zero_()), "layer", None, (g_x,), ("y", "w_post"))):
        want = grads(lambda c, out: None, post, pre, seeds, names)
        got = grads(change, post, pre, seeds, names)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for change, names in ((lambda c, out: out[0].detach().zero_(), ("x",)), (lambda c, out: c["x"].zero_(), ("scale",)),
                          (lambda c, out: c["y"].zero_(), ("gate",))):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            grads(change, "rms", "rms", (g_x, g_h), names)


@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.to(torch.float64), lambda t: t[..., :1].contiguous(),
                                    lambda t: t.flatten()[:1], lambda t: t[None]])
def test_hooks_that_hand_back_something_else(change):
    """Refused on the host, whichever of the saved tensors it is; the same values at another address are taken."""
    t, g_x, g_h = _operands("element", F32)
    n = len(_saved(_learn(t, NAMES), "rms", "layer")[0])
    assert n == 9                       # x, y, three of the vectors and post's bias, gate, x', statistics
    for which in range(n):
        c, seen = _learn(t, NAMES), []

        def pack(v):
            seen.append(v)
            return len(seen) - 1, v
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda p: change(p[1]) if p[0] == which else p[1].clone()):
            out = _call(c, "rms", "layer")
            with pytest.raises((RuntimeError, ValueError, TypeError)):
                torch.autograd.grad(out, [c[k] for k in NAMES], (g_x, g_h))
                pytest.fail(str(which))
    want = _learn(t, NAMES)
    want = torch.autograd.grad(_call(want, "rms", "layer"), [want[k] for k in NAMES], (g_x, g_h))
    c = _learn(t, NAMES)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: v.T.contiguous().T if v.dim() == 2 else v.clone()):
        got = torch.autograd.grad(_call(c, "rms", "layer"), [c[k] for k in NAMES], (g_x, g_h))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
