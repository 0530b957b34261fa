"""The weighted sum of a plan at the C entry points on the CPU: what it refuses, on the host and before anything is enqueued."""
import ctypes as C

import pytest
from test_experts_abi import BF, F32, FAKE, Experts, _of, _refused

from bitsparse_amd import _lib

PLAN = dict(rows=8, tokens=4, experts=4, top_k=2, offsets=FAKE)


def _forward(plan={}, y=FAKE, y_type=BF, y_stride=64, w=FAKE, place=FAKE, cols=64, out=FAKE):
    e = _of(Experts, PLAN, plan)
    return _lib.load().bs_expert_combine_plan(C.byref(e), y, y_type, y_stride, w, place, cols, out, None)


def _backward(plan={}, g=FAKE, g_stride=64, y=FAKE, y_stride=64, w=FAKE, place=FAKE, cols=64, dy=FAKE, dw=FAKE):
    e = _of(Experts, PLAN, plan)
    return _lib.load().bs_expert_combine_plan_backward(C.byref(e), g, g_stride, y, y_stride, w, place, cols, dy, dw, None)


@pytest.mark.parametrize("plan,word", [(dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(offsets=None), "offsets"),
                                       (dict(offsets=FAKE + 2), "offsets"), (dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(tokens=-1), "tokens"),
                                       (dict(rows=1 << 31), "2^31")])
def test_plan_refusals(plan, word):
    _refused(_forward(plan), word)
    _refused(_backward(plan), word)


def test_operand_refusals():
    for kw, word in [(dict(y=None), "null"), (dict(place=None), "null"), (dict(out=None), "null"), (dict(y_stride=-1), "stride"), (dict(y=FAKE + 1), "misaligned"),
                     (dict(y=FAKE + 2, y_type=F32), "misaligned"), (dict(w=FAKE + 2), "misaligned"), (dict(y_type=1), "dtype"), (dict(cols=1 << 40), "2^40")]:
        _refused(_forward(**kw), word)
    for kw, word in [(dict(g=None), "null"), (dict(place=None), "null"), (dict(y=None), "null"), (dict(g_stride=-1), "stride"),
                     (dict(dy=FAKE + 1), "misaligned"), (dict(dw=FAKE + 2), "misaligned"), (dict(cols=1 << 40), "2^40")]:
        _refused(_backward(**kw), word)
    _refused(_lib.load().bs_expert_combine_plan(None, FAKE, BF, 64, FAKE, FAKE, 64, FAKE, None), "null")
    _refused(_lib.load().bs_expert_combine_plan_backward(None, FAKE, 64, FAKE, 64, FAKE, FAKE, 64, FAKE, FAKE, None), "null")
    assert _forward(dict(tokens=0), place=None) == _forward(cols=0, y=None) == _backward(dy=None, dw=None) == _lib.BS_OK
