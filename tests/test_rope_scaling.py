"""CPU tests of RopeCache's scalings against the formulas in 64 bits: a table
value is the formula's rounded once (2^-24 of its size; the angles' own error, at
most 2^-50 of one of up to 2^17 radians, is far below)."""
import math

import numpy as np
import pytest

from cpuforge_amd import CfattnError, LinearScaling, Llama3Scaling, NtkScaling, RopeCache, YarnScaling


def table(inv, max_pos, size=1.0):
    angle = np.arange(max_pos, dtype=np.float64)[:, None] * inv
    return np.cos(angle) * size, np.sin(angle) * size


def plain(dim, theta):
    return theta ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)


def check(rope, inv, size=1.0):
    for got, want in zip((rope.cos, rope.sin), table(inv, rope.max_pos, size)):
        assert got.shape == want.shape
        assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -32)


@pytest.mark.parametrize("dim", [2, 10, 64, 128])
def test_linear_and_ntk(dim):
    check(RopeCache(dim, 3000, 1e4, LinearScaling(4.0)), plain(dim, 1e4) / 4)
    inv = plain(dim, 1e4 * 8.0 ** (dim / (dim - 2)) if dim > 2 else 1e4)
    check(RopeCache(dim, 3000, 1e4, NtkScaling(8.0)), inv)
    if dim > 2:  # the slowest pair turns 8 times slower, the fastest as before
        slowest = plain(dim, 1e4)[-1] / 8
        assert inv[0] == 1.0 and abs(inv[-1] - slowest) <= 1e-12 * slowest


@pytest.mark.parametrize("dim,theta,factor,trained", [(64, 1e4, 8.0, 4096), (128, 1e6, 4.0, 32768), (16, 1e4, 32.0, 100),
                                                      (2, 1e4, 4.0, 64)])
@pytest.mark.parametrize("attention", [None, 1.0, 0.7])
def test_yarn(dim, theta, factor, trained, attention):
    rope = RopeCache(dim, 2000, theta, YarnScaling(factor, trained, attention_factor=attention))
    inv = plain(dim, theta)
    turns = [dim * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (32.0, 1.0)]
    lo, hi = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), dim - 1)
    slow = np.clip((np.arange(dim // 2) - lo) / (hi - lo if hi > lo else 1e-3), 0, 1)
    size = 0.1 * math.log(factor) + 1 if attention is None else attention
    check(rope, inv * (1 - slow) + inv / factor * slow, size)
    # Pairs that turn often are as they were, those that hardly turn slowed down whole.
    if dim == 64:
        assert slow[0] == 0 and slow[-1] == 1


def test_plain_and_llama3_tables_are_the_same_as_before():
    sc = Llama3Scaling(32.0, 1.0, 4.0, 8192.0)
    inv = np.array([sc.apply(f) for f in plain(64, 5e5)])
    check(RopeCache(64, 500, 5e5, sc), inv)
    check(RopeCache(64, 500, 5e5), plain(64, 5e5))


@pytest.mark.parametrize("scaling", [LinearScaling(0.0), NtkScaling(-1.0), LinearScaling(float("nan")),
                                     YarnScaling(4.0, 0), YarnScaling(4.0, 64, beta_fast=1.0, beta_slow=2.0),
                                     YarnScaling(4.0, 64, beta_slow=0.0)])
def test_refusals(scaling):
    with pytest.raises(CfattnError):
        RopeCache(64, 10, 1e4, scaling)


def test_refused_attention_factor():
    with pytest.raises(ValueError):
        RopeCache(64, 10, 1e4, YarnScaling(4.0, 64, attention_factor=-1.0))
