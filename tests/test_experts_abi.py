"""The experts' and dropout's C entry points on the CPU: what they refuse, on the host and before anything is enqueued."""
import ctypes as C

import pytest

from bitsparse_amd import _lib

FAKE = 0x10000      # never dereferenced: the checks fail first
BF, F32 = 0, 3


class Drop(C.Structure):
    _fields_ = [("seed", C.c_uint64), ("offset", C.c_uint64), ("state", C.c_void_p), ("below", C.c_int)]


class Route(C.Structure):
    _fields_ = [("tokens", C.c_int64), ("experts", C.c_int), ("top_k", C.c_int), ("logits", C.c_void_p), ("logits_type", C.c_int),
                ("logits_stride", C.c_int64), ("bias", C.c_void_p), ("score", C.c_int), ("groups", C.c_int), ("top_groups", C.c_int),
                ("group_best", C.c_int), ("renormalize", C.c_int), ("scale", C.c_float)]


class Experts(C.Structure):
    _fields_ = [("rows", C.c_int64), ("tokens", C.c_int64), ("experts", C.c_int), ("top_k", C.c_int), ("offsets", C.c_void_p), ("order", C.c_void_p)]


def _refused(rc, word):
    assert rc == _lib.BS_ERR_INVALID
    assert word in _lib.load().bs_last_error().decode(), _lib.load().bs_last_error()


def _of(cls, base, kw):
    a = cls(**base)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("drop,kw,word", [
    (dict(below=-1), {}, "below"), (dict(below=65537), {}, "below"), (dict(state=FAKE + 4), {}, "state"), ({}, dict(type=1), "dtype"),
    ({}, dict(rows=-1), "rows"), ({}, dict(rows=1 << 32), "2^32"), ({}, dict(cols=1 << 32), "2^32"), ({}, dict(rows=1 << 30, cols=1 << 20), "2^40"),
    ({}, dict(x=None), "null"), ({}, dict(out=None), "null"), ({}, dict(stride=-1), "stride"), ({}, dict(x=FAKE + 1), "misaligned"),
    ({}, dict(out=FAKE + 2, type=F32), "misaligned")])
def test_dropout_refusals(drop, kw, word):
    L = _lib.load()
    a = dict(x=FAKE, type=BF, rows=4, cols=8, stride=8, out=FAKE)
    a.update(kw)
    d = _of(Drop, dict(below=100), drop)
    _refused(L.bs_dropout(C.byref(d), a["x"], a["type"], a["rows"], a["cols"], a["stride"], a["out"], None), word)


def test_dropout_of_nothing():
    L = _lib.load()
    d = Drop(below=1)
    assert L.bs_dropout(C.byref(d), None, BF, 0, 8, 8, None, None) == _lib.BS_OK
    assert L.bs_dropout(C.byref(d), None, BF, 8, 0, 0, None, None) == _lib.BS_OK
    _refused(L.bs_dropout(None, FAKE, BF, 4, 8, 8, FAKE, None), "null")


def test_join_with_dropout_refusals():
    from test_step_abi import JoinGrads, _join
    L = _lib.load()
    ok = _join(stats_post=FAKE, stats_pre=FAKE)
    g = JoinGrads(x1=FAKE, grad_x1=FAKE, grad_h=FAKE)
    for a, d, word in [(ok, None, "null drop"), (ok, Drop(below=-3), "below"), (_join(y=None, norm_post=0, stats_pre=FAKE), Drop(below=3), "needs y"),
                       (_join(rows=1 << 32, cols=8, x_stride=8, y_stride=8), Drop(below=3), "2^32"), (_join(norm_pre=3), Drop(below=3), "norm")]:
        _refused(L.bs_join_drop_forward(C.byref(a), d and C.byref(d), FAKE, FAKE, None), word)
        _refused(L.bs_join_drop_backward(C.byref(a), C.byref(g), d and C.byref(d), FAKE, 1 << 40, None), word)
    _refused(L.bs_join_drop_forward(C.byref(ok), C.byref(Drop(below=3)), None, FAKE, None), "null result")


ROUTE = dict(tokens=4, experts=16, top_k=2, logits=FAKE, logits_type=F32, logits_stride=16, groups=1, top_groups=1, group_best=1, scale=1.0)
ROUTE_BAD = [(dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(top_k=0), "top_k"), (dict(top_k=17), "top_k"),
             (dict(experts=100, top_k=65), "top_k"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30), "2^31"), (dict(tokens=1 << 62, experts=4), "2^31"), (dict(logits_type=1), "dtype"),
             (dict(score=2), "score"), (dict(groups=0), "groups"), (dict(groups=3), "groups"), (dict(experts=1024, groups=128), "groups"),
             (dict(groups=4, top_groups=5), "top_groups"), (dict(groups=4, top_groups=0), "top_groups"), (dict(group_best=3), "group_best"),
             (dict(groups=8, top_groups=1, top_k=3), "more than"), (dict(logits_stride=-1), "stride"), (dict(logits=None), "null"),
             (dict(logits=FAKE + 2), "misaligned"), (dict(bias=FAKE + 1), "misaligned")]


@pytest.mark.parametrize("bad,word", ROUTE_BAD)
def test_route_refusals(bad, word):
    L = _lib.load()
    a = _of(Route, ROUTE, bad)
    _refused(L.bs_route_forward(C.byref(a), FAKE, FAKE, None), word)
    _refused(L.bs_route_backward(C.byref(a), FAKE, FAKE, FAKE, None), word)


def test_route_results_and_plan():
    L = _lib.load()
    a = _of(Route, ROUTE, {})
    _refused(L.bs_route_forward(None, FAKE, FAKE, None), "null")
    for args in ((None, FAKE), (FAKE, None), (FAKE + 2, FAKE), (FAKE, FAKE + 1)):
        _refused(L.bs_route_forward(C.byref(a), *args, None), "result")
    for args in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None), (FAKE, FAKE, FAKE + 2)):
        _refused(L.bs_route_backward(C.byref(a), *args, None), "operand")
    none = _of(Route, ROUTE, dict(tokens=0, logits=None))
    assert L.bs_route_forward(C.byref(none), None, None, None) == _lib.BS_OK
    assert L.bs_route_backward(C.byref(none), None, None, None, None) == _lib.BS_OK
    need = L.bs_expert_plan_workspace_bytes
    assert need(0, 8) == need(100, 8) == need(100, 0) == need(100, 2000) == 0 < need(100000, 8)
    for args, word in [((FAKE, 10, 0, FAKE, FAKE, FAKE, None, 0), "experts"), ((FAKE, 10, 1025, FAKE, FAKE, FAKE, None, 0), "experts"),
                       ((FAKE, -1, 4, FAKE, FAKE, FAKE, None, 0), "pairs"), ((FAKE, 1 << 31, 4, FAKE, FAKE, FAKE, None, 0), "pairs"),
                       ((None, 10, 4, FAKE, FAKE, FAKE, None, 0), "null"), ((FAKE, 10, 4, None, FAKE, FAKE, None, 0), "null"),
                       ((FAKE, 10, 4, FAKE, FAKE + 2, FAKE, None, 0), "misaligned"), ((FAKE, 100000, 4, FAKE, FAKE, FAKE, None, 0), "workspace"),
                       ((FAKE, 100000, 4, FAKE, FAKE, FAKE, FAKE, need(100000, 4) - 1), "workspace")]:
        _refused(L.bs_expert_plan(*args, None), word)


def _products(experts, kw):
    """The three calls with the same operands"""
    L = _lib.load()
    e = _of(Experts, dict(rows=32, tokens=16, experts=4, top_k=2, offsets=FAKE), experts)
    a = dict(x=FAKE, x_stride=64, W=FAKE, w_stride=64, inn=64, out=64, y=FAKE)
    a.update(kw)
    at = C.byref(e)
    return (lambda: L.bs_expert_linear(at, a["x"], a["x_stride"], a["W"], a["w_stride"], a["inn"], a["out"], 0, 1.0, a["y"], None),
            lambda: L.bs_expert_linear_dx(at, a["x"], a["x_stride"], a["W"], a["w_stride"], a["inn"], a["out"], a["y"], BF, None),
            lambda: L.bs_expert_linear_dw(at, a["x"], a["x_stride"], a["W"], a["w_stride"], a["inn"], a["out"], a["y"], None))


@pytest.mark.parametrize("experts,kw,word", [
    (dict(experts=0), {}, "experts"), (dict(experts=1025), {}, "experts"), (dict(rows=-1), {}, "rows"), (dict(rows=1 << 31), {}, "rows"),
    (dict(tokens=1 << 31), {}, "tokens"), (dict(top_k=0), {}, "top_k"), ({}, dict(inn=0), "in and out"), ({}, dict(out=65537), "in and out"),
    ({}, dict(inn=65536, out=65536), "2^30"), (dict(offsets=None), {}, "offsets"), (dict(offsets=FAKE + 2), {}, "offsets"),
    ({}, dict(x=None), "null"), ({}, dict(x=FAKE + 8), "16-byte"), ({}, dict(x_stride=60), "16-byte"), ({}, dict(x_stride=56), "16-byte"),
    ({}, dict(x_stride=1 << 22), "2^22"), ({}, dict(W=None), "null"), ({}, dict(w_stride=72 - 4), "16-byte"), ({}, dict(y=None), "misaligned"),
    ({}, dict(y=FAKE + 4), "misaligned")])
def test_product_refusals(experts, kw, word):
    for call in _products(experts, kw):
        _refused(call(), word)


def test_products_and_order():
    forward, dx, dw = _products(dict(order=FAKE), {})
    _refused(dx(), "order")
    _refused(dw(), "order")
    forward, _, _ = _products(dict(order=FAKE, tokens=(1 << 31) - 1), {})
    _refused(forward(), "4 GiB")
    forward, _, _ = _products({}, dict(w_stride=1 << 20, out=4096))
    _refused(forward(), "4 GiB")
    # 2^31 / 256 tiles of rows, of which any size of tile has two or more over the columns
    forward, _, _ = _products(dict(rows=(1 << 31) - 1), dict(x_stride=8, w_stride=8, inn=8, out=264))
    _refused(forward(), "tiles")
    L = _lib.load()
    e = Experts(rows=32, tokens=16, experts=4, top_k=2, offsets=FAKE)
    _refused(L.bs_expert_linear(C.byref(e), FAKE, 64, FAKE, 64, 64, 64, 3, 1.0, FAKE, None), "activation")
    _refused(L.bs_expert_linear_dx(C.byref(e), FAKE, 64, FAKE, 64, 64, 64, FAKE, 2, None), "dtype")
    _refused(L.bs_expert_linear(None, FAKE, 64, FAKE, 64, 64, 64, 0, 1.0, FAKE, None), "null")
    e.rows = 0
    assert L.bs_expert_linear(C.byref(e), None, 64, FAKE, 64, 64, 64, 0, 1.0, None, None) == _lib.BS_OK
    assert L.bs_expert_linear_dx(C.byref(e), None, 64, FAKE, 64, 64, 64, None, BF, None) == _lib.BS_OK


@pytest.mark.parametrize("args,word", [
    ((FAKE, -1, 8, 8, FAKE, 8), "width"), ((FAKE, 4, 9, 9, FAKE, 8), "width"), ((FAKE, 4, 5, 5, FAKE, 12), "width"), ((FAKE, 4, 5, -5, FAKE, 8), "width"),
    ((None, 4, 5, 5, FAKE, 8), "null"), ((FAKE, 4, 5, 5, None, 8), "null"), ((FAKE + 1, 4, 5, 5, FAKE, 8), "misaligned"), ((FAKE, 4, 5, 5, FAKE + 8, 8), "misaligned")])
def test_pad_refusals(args, word):
    _refused(_lib.load().bs_pad_rows(*args, None), word)


def test_sum_refusals():
    L = _lib.load()

    def forward(y=FAKE, y_type=BF, y_stride=64, w=FAKE, place=FAKE, tokens=4, k=2, rows=8, cols=64, out=FAKE):
        return L.bs_expert_combine(y, y_type, y_stride, w, place, tokens, k, rows, cols, out, None)

    def backward(g=FAKE, g_stride=64, y=FAKE, y_stride=64, w=FAKE, place=FAKE, used=FAKE, tokens=4, k=2, rows=8, cols=64, dy=FAKE, dw=FAKE):
        return L.bs_expert_combine_backward(g, g_stride, y, y_stride, w, place, used, tokens, k, rows, cols, dy, dw, None)

    def between(g=FAKE, r=FAKE, rows=8, cols=64, w=FAKE, order=FAKE, used=FAKE, pairs=8, dw=FAKE):
        return L.bs_experts_act_grad(g, r, rows, cols, 1, 1.0, w, order, used, pairs, dw, None)
    for kw, word in [(dict(k=0), "top_k"), (dict(k=65), "top_k"), (dict(tokens=-1), "tokens"), (dict(rows=1 << 31), "2^31"), (dict(rows=1 << 30, cols=1 << 20), "2^40")]:
        _refused(forward(**kw), word)
        _refused(backward(**kw), word)
    for kw, word in [(dict(y=None), "null"), (dict(place=None), "null"), (dict(out=None), "null"), (dict(y_stride=-1), "stride"), (dict(y=FAKE + 1), "misaligned"),
                     (dict(y=FAKE + 2, y_type=F32), "misaligned"), (dict(w=FAKE + 2), "misaligned"), (dict(y_type=1), "dtype")]:
        _refused(forward(**kw), word)
    for kw, word in [(dict(g=None), "null"), (dict(place=None), "null"), (dict(used=None), "null"), (dict(y=None), "null"), (dict(g_stride=-1), "stride"),
                     (dict(dy=FAKE + 1), "misaligned"), (dict(dw=FAKE + 2), "misaligned")]:
        _refused(backward(**kw), word)
    for kw, word in [(dict(rows=-1), "rows"), (dict(pairs=-1), "rows"), (dict(g=None), "null"), (dict(r=None), "null"), (dict(w=None), "null"), (dict(order=None), "null"),
                     (dict(used=None), "null"), (dict(g=FAKE + 1), "misaligned"), (dict(dw=FAKE + 1), "misaligned")]:
        _refused(between(**kw), word)
    assert forward(tokens=0, place=None) == backward(dy=None, dw=None) == between(rows=0, g=None) == _lib.BS_OK
