"""bs_join_* and bs_newton_schulz on the CPU: what they refuse, on the host and before anything is enqueued."""
import ctypes as C

import pytest

from bitsparse_amd import _lib

FAKE = 0x10000      # never dereferenced: the checks fail first
BF, F32 = 0, 3


class Vector(C.Structure):
    _fields_ = [("data", C.c_void_p), ("type", C.c_int)]


class JoinArgs(C.Structure):
    _fields_ = [("rows", C.c_int64), ("cols", C.c_int64), ("x_type", C.c_int), ("y_type", C.c_int), ("norm_post", C.c_int),
                ("norm_pre", C.c_int), ("eps_post", C.c_float), ("eps_pre", C.c_float), ("x", C.c_void_p), ("y", C.c_void_p),
                ("x_stride", C.c_int64), ("y_stride", C.c_int64), ("weight_post", Vector), ("bias_post", Vector),
                ("weight_pre", Vector), ("bias_pre", Vector), ("gate", Vector), ("scale", Vector), ("gate_per", C.c_int),
                ("scale_per", C.c_int), ("gate_stride", C.c_int64), ("scale_value", C.c_float), ("stats_post", C.c_void_p),
                ("stats_pre", C.c_void_p)]


class JoinGrads(C.Structure):
    _fields_ = [("x1", C.c_void_p), ("grad_x1", C.c_void_p), ("grad_h", C.c_void_p), ("grad_x1_stride", C.c_int64),
                ("grad_h_stride", C.c_int64)] + [(n, C.c_void_p) for n in (
                    "d_x", "d_y", "d_gate", "d_scale", "d_weight_post", "d_bias_post", "d_weight_pre", "d_bias_pre")]


class Matrix(C.Structure):
    _fields_ = [("grad", C.c_void_p), ("momentum", C.c_void_p), ("out", C.c_void_p), ("grad_stride", C.c_int64),
                ("momentum_stride", C.c_int64), ("out_stride", C.c_int64), ("transposed", C.c_int)]


class Rule(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("grad_type", "momentum_type", "out_type", "momentum", "nesterov", "update", "precise",
                                       "steps")] + [(n, C.c_float) for n in ("a", "b", "c", "eps", "mu", "keep", "rate")]


def _join(**kw):
    a = JoinArgs(rows=4, cols=64, norm_post=1, norm_pre=1, x=FAKE, y=FAKE, x_stride=64, y_stride=64, scale_value=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _refused(rc, word):
    assert rc == _lib.BS_ERR_INVALID
    assert word in _lib.load().bs_last_error().decode(), _lib.load().bs_last_error()


JOIN_BAD = [(dict(cols=0), "cols"), (dict(cols=32769), "cols"), (dict(rows=-1), "rows"), (dict(rows=1 << 39), "2^40"),
            (dict(x_type=1), "dtypes"), (dict(y_type=F32), "dtypes"), (dict(norm_pre=3), "norm"), (dict(y=None, norm_post=0, norm_pre=0), "neither"),
            (dict(y=None), "need y"), (dict(x=None), "null x"), (dict(x_stride=-1), "stride"), (dict(x=FAKE + 1), "misaligned"),
            (dict(weight_pre=Vector(FAKE, 2)), "vector"), (dict(weight_pre=Vector(FAKE + 2, F32)), "vector"),
            (dict(norm_post=0, weight_post=Vector(FAKE, BF)), "without norm_post"), (dict(norm_pre=0, bias_pre=Vector(FAKE, BF)), "without norm_pre"),
            (dict(gate=Vector(FAKE, BF)), "gate_per"), (dict(gate_per=2), "gate_per"), (dict(scale=Vector(FAKE, BF), scale_per=3), "scale_per"),
            (dict(stats_pre=FAKE + 4), "stats")]


@pytest.mark.parametrize("bad,word", JOIN_BAD)
def test_join_refusals(bad, word):
    L = _lib.load()
    a = _join(**bad)
    _refused(L.bs_join_forward(C.byref(a), FAKE, FAKE, None), word)
    g = JoinGrads(x1=FAKE, grad_x1=FAKE, grad_h=FAKE)
    _refused(L.bs_join_backward(C.byref(a), C.byref(g), FAKE, 1 << 30, None), word)


def test_join_results_and_gradients():
    L = _lib.load()
    ok = _join()
    _refused(L.bs_join_forward(None, FAKE, FAKE, None), "null")
    _refused(L.bs_join_forward(C.byref(ok), None, FAKE, None), "null result")
    _refused(L.bs_join_forward(C.byref(ok), FAKE, FAKE + 1, None), "misaligned")
    assert L.bs_join_forward(C.byref(_join(rows=0)), None, None, None) == _lib.BS_OK
    full = dict(stats_post=FAKE, stats_pre=FAKE)
    for args, grads, word in [
            (_join(**full), None, "null"), (_join(**full), JoinGrads(x1=FAKE), "no gradient"),
            (_join(rows=0), JoinGrads(x1=FAKE, grad_h=FAKE), "no rows"), (_join(), JoinGrads(x1=FAKE, grad_h=FAKE), "statistics"),
            (_join(**full), JoinGrads(grad_h=FAKE), "x1"), (_join(**full), JoinGrads(x1=FAKE, grad_h=FAKE, grad_h_stride=-1), "stride"),
            (_join(**full), JoinGrads(x1=FAKE, grad_h=FAKE, d_weight_pre=FAKE), "absent vector"),
            (_join(**full), JoinGrads(x1=FAKE, grad_h=FAKE, d_x=FAKE + 1), "misaligned"),
            (_join(norm_pre=0, stats_post=FAKE), JoinGrads(grad_h=FAKE), "without norm_pre"),
            (_join(y=None, norm_post=0, stats_pre=FAKE), JoinGrads(grad_h=FAKE, d_y=FAKE), "need y")]:
        _refused(L.bs_join_backward(C.byref(args), grads and C.byref(grads), FAKE, 1 << 30, None), word)
    g = JoinGrads(x1=FAKE, grad_h=FAKE)
    need = L.bs_join_backward_workspace_bytes(4, 64)
    assert need > 0 and L.bs_join_backward_workspace_bytes(0, 64) == 0
    _refused(L.bs_join_backward(C.byref(_join(**full)), C.byref(g), FAKE, need - 1, None), "workspace")
    _refused(L.bs_join_backward(C.byref(_join(**full)), C.byref(g), None, need, None), "workspace")


def _schulz(matrix=None, rule=None, count=1, rows=8, cols=12, ws=FAKE, nbytes=1 << 40):
    m = Matrix(grad=FAKE, out=FAKE, momentum=FAKE, grad_stride=12, out_stride=12, momentum_stride=12)
    for k, v in (matrix or {}).items():
        setattr(m, k, v)
    r = Rule(grad_type=BF, momentum_type=F32, out_type=BF, steps=5, momentum=1)
    for k, v in (rule or {}).items():
        setattr(r, k, v)
    return _lib.load().bs_newton_schulz(C.byref(m), count, rows, cols, C.byref(r), ws, nbytes, None)


@pytest.mark.parametrize("kw,word", [
    (dict(count=-1), "count"), (dict(rows=0), "rows"), (dict(cols=65537), "65536"), (dict(rows=32768, cols=32768), "2^29"),
    (dict(rule=dict(steps=0)), "steps"), (dict(rule=dict(steps=101)), "steps"), (dict(rule=dict(grad_type=1)), "dtypes"),
    (dict(rule=dict(momentum_type=7)), "dtypes"), (dict(rule=dict(out_type=2)), "dtypes"), (dict(matrix=dict(grad=None)), "null"),
    (dict(matrix=dict(momentum=None)), "null"), (dict(matrix=dict(momentum=FAKE + 2)), "misaligned"), (dict(matrix=dict(out=FAKE + 1)), "misaligned"),
    (dict(matrix=dict(out_stride=11)), "overlap"), (dict(matrix=dict(momentum_stride=3)), "overlap"), (dict(matrix=dict(grad_stride=-1)), "overlap"),
    (dict(ws=None), "workspace"), (dict(ws=FAKE + 8), "workspace"), (dict(nbytes=100), "workspace")])
def test_newton_schulz_refusals(kw, word):
    _refused(_schulz(**kw), word)


@pytest.mark.parametrize("a,b,c,steps,ok", [
    (3.4445, -4.7750, 2.0315, 100, True), (1.5, -0.5, 0.0, 100, True), (2.0, -1.5, 0.5, 5, True),
    (3.0, 0.0, 0.0, 2, True), (3.0, 0.0, 0.0, 3, False),            # X of 1, 3 and 9, A of 1, 9 and 81
    (4.5, 0.0, 0.0, 1, True), (4.5, 0.0, 0.0, 2, False),            # the last X is no operand; A of 1 and 20.25
    (14.9, 0.0, 0.0, 1, True), (15.1, 0.0, 0.0, 1, False), (-15.1, 0.0, 0.0, 1, False), (0.0, 0.0, 16.0, 1, False),
    (0.0, 70.0, -70.0, 1, False),                                   # B is largest inside the range, 17.5 at t = 0.5
    (-10.0, 20.0, 0.0, 1, False), (-7.0, 14.0, 0.0, 1, True),       # b X + c A X
    (float("nan"), 0.0, 0.0, 1, False), (0.0, float("inf"), 0.0, 1, False)])
def test_newton_schulz_range(a, b, c, steps, ok):
    """Coefficients whose operands fp16 does not hold; what is held gets as far as the workspace."""
    _refused(_schulz(rule=dict(a=a, b=b, c=c, steps=steps), ws=None), "workspace" if ok else "range")


def test_newton_schulz_workspace():
    L = _lib.load()
    assert _schulz(count=0) == _lib.BS_OK
    one = L.bs_newton_schulz_workspace_bytes(256, 1024, 1, 0)
    # X twice, A and B, with padding; a transposed shape the same; precise operands twice that
    assert 2 * 2 * 256 * 1024 + 2 * 2 * 256 * 256 < one == L.bs_newton_schulz_workspace_bytes(1024, 256, 1, 0)
    assert one < L.bs_newton_schulz_workspace_bytes(256, 1024, 1, 1) < 2 * one + 1
    assert L.bs_newton_schulz_workspace_bytes(0, 4, 1, 0) == 0
    # what goes together is bounded: more matrices take no more room
    assert L.bs_newton_schulz_workspace_bytes(256, 1024, 64, 0) == L.bs_newton_schulz_workspace_bytes(256, 1024, 1000, 0)
