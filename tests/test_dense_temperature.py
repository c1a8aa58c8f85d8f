"""The loss's temperature is a factor of everything: one whose square is no float above zero is refused, not answered with NaN."""
import pytest

from tests.test_dense_native import INVALID, P, WORKSPACE, lib  # noqa: F401


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), float("inf"), 1e20, 1e-23, 1e-39])
def test_temperatures_refused(lib, temperature):
    assert lib.geo_sc_distill_topk(P, 1, 10, P, 1, P, 4, 5, 10, 3, temperature, 2, P, P, P, 1 << 20, None) == INVALID
    assert lib.geo_sc_distill_topk_backward(P, 2, P, 1, 10, P, 1, P, 4, 5, 10, 3, temperature, P, P, None) == INVALID


@pytest.mark.parametrize("temperature", [1e-22, 1e-3, 1.0, 1e19])
def test_temperatures_taken(lib, temperature):
    # (as far as the next check)
    assert lib.geo_sc_distill_topk(P, 1, 10, P, 1, P, 4, 5, 10, 3, temperature, 2, P, P, None, 0, None) == WORKSPACE
