"""Rotary frequencies over the whole range of theta: the plan holds turns per
position in 2^-64 turns, so a frequency has to lie below one turn."""
import math

import numpy as np
import pytest

from tests.test_token_ops_cpu import _lib, _rot


@pytest.mark.parametrize("theta", [1e-3, 1e-12, 1e-300, 0.1])
@pytest.mark.parametrize("freq", [0, 1])
def test_frequencies_of_more_than_a_turn_are_refused(theta, freq):
    """Their fraction of a turn would keep only the bits that the whole turns leave:
    2^-28 turns per position at theta = 1e-12, an eighth of a turn at position 2^25."""
    L = _lib()
    plan = L.RotaryPlan()
    assert L.lib.ie_rotary_plan_init(_rot(L, theta=theta, freq=freq), plan) == L.IE_UNSUPPORTED
    assert b"turn" in L.lib.ie_cuda_last_error()


@pytest.mark.parametrize("theta", [0.2, 0.5, 1.0, 1.5, 1e4, 1e6, 1e300])
@pytest.mark.parametrize("freq", [0, 1])
def test_frequencies_below_a_turn(theta, freq):
    """As test_rotary_plan_frequencies: 2^-65 for the fixed point and 2^-64 relative for
    the power, against 2 math.pi of 53 bits."""
    L = _lib()
    plan = L.RotaryPlan()
    assert L.lib.ie_rotary_plan_init(_rot(L, theta=theta, freq=freq), plan) == 0
    for i in range(32):
        e = np.longdouble(i) / 32 if freq == 0 else np.longdouble(i % 16) / 16
        f = np.longdouble(theta) ** -e / (2 * np.longdouble(math.pi))
        assert f < 1
        assert abs(float(plan.turns[i]) * 2.0 ** -64 - float(f)) <= 2.0 ** -52 * float(f) + 2.0 ** -63
