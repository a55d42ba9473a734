"""CPU tests of RopeCache's scalings at the ends of their parameters' ranges."""
import math

import numpy as np
import pytest

from cpuforge_amd import CfattnError, LinearScaling, NtkScaling, RopeCache, YarnScaling

INF = float("inf")


def tables(rope):
    return np.stack([rope.cos, rope.sin])


def test_a_yarn_factor_below_one_needs_a_size():
    """0.1 ln(factor) + 1 is of longer contexts: below 1 it shrinks the scores, and it is
    negative from e^-10 on."""
    for factor in (0.999, 0.5, math.exp(-11)):
        with pytest.raises(CfattnError):
            RopeCache(64, 10, 1e4, YarnScaling(factor, 64))
        rope = RopeCache(64, 10, 1e4, YarnScaling(factor, 64, attention_factor=1.0))
        assert np.all(rope.cos[0] == 1.0) and np.all(rope.sin[0] == 0.0)
    assert np.array_equal(tables(RopeCache(64, 10, 1e4, YarnScaling(1.0, 64))), tables(RopeCache(64, 10, 1e4)))


@pytest.mark.parametrize("scaling", [LinearScaling(INF), NtkScaling(INF), NtkScaling(1e300), YarnScaling(INF, 64),
                                     YarnScaling(4.0, INF), YarnScaling(4.0, 64, beta_fast=INF),
                                     YarnScaling(4.0, 64, attention_factor=INF)])
def test_values_that_are_not_finite_are_refused(scaling):
    with pytest.raises(CfattnError):
        RopeCache(64, 10, 1e4, scaling)


def test_a_base_that_is_not_finite_is_refused():
    for theta in (INF, float("nan"), 0.0):
        with pytest.raises(CfattnError):
            RopeCache(64, 10, theta, LinearScaling(2.0))
