"""What bs_newton_schulz refuses of its rule, on the host."""
import pytest

from tests.test_step_abi import _refused, _schulz


@pytest.mark.parametrize("eps,ok", [(0.0, True), (1e-7, True), (float("inf"), True), (-1e-7, False), (-1.0, False), (float("nan"), False)])
def test_eps(eps, ok):
    _refused(_schulz(rule=dict(eps=eps, a=3.4445, b=-4.775, c=2.0315), ws=None), "workspace" if ok else "eps")
