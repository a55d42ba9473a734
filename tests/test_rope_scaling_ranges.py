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


@pytest.mark.parametrize("trained", [1.0, 4.0, 6.0, 2 * math.pi])
@pytest.mark.parametrize("dim", [2, 10, 64])
def test_every_pair_of_a_short_context_is_slow(dim, trained):
    """The first pair turns once in 2 pi positions: in fewer no pair turns more than
    beta_slow = 1 times, and all are `factor` times slower."""
    got = RopeCache(dim, 50, 1e4, YarnScaling(4.0, trained, attention_factor=1.0))
    assert np.array_equal(tables(got), tables(RopeCache(dim, 50, 1e4, LinearScaling(4.0))))


def test_every_pair_of_a_long_context_is_fast():
    got = RopeCache(64, 50, 1e4, YarnScaling(4.0, 1e9, attention_factor=1.0))
    assert np.array_equal(tables(got), tables(RopeCache(64, 50, 1e4)))
