"""GPU tests that cfops_adamw8_pack_multi rounds every moment to the nearest of its
steps (include/cfops.h, cfops_adamw_tensor)."""
import numpy as np
import pytest
import torch

from tests import adamw8_ref as R
from tests.test_gpu_adamw8 import dev, moments

pytestmark = pytest.mark.gpu


def packed(m, v):
    from cpuforge_amd import ops as P
    d = dict(m=dev(m), v=dev(v), state8=P.adamw8_state(m.size))
    P.adamw8_pack_multi([d])
    return moments(d)


def test_either_side_of_a_middle():
    """The neighbours in f32 of the middles between 1, 1.125, .. 2: below it down, at
    it and above it up, for m of either sign and for v."""
    steps = 1 + np.arange(8) / 8
    mid = (steps + 1 / 16).astype(np.float32)
    below, above = np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(9))
    x = np.concatenate([below, mid, above, [2.0]]).astype(np.float64)
    want = np.concatenate([steps, steps + 0.125, steps + 0.125, [2.0]])
    for sign in (1, -1):
        m, v = packed(sign * x, x)
        assert np.array_equal(m, sign * want) and np.array_equal(v, want)
    # Some way off the middle, at the 17 bits that a rounding looks at.
    for k in range(1, 9):
        x = np.concatenate([steps + (0.5 - k * 2.0 ** -17) / 8, [2.0]])
        m, v = packed(x, x)
        assert np.array_equal(m, np.concatenate([steps, [2.0]])) and np.array_equal(v, np.concatenate([steps, [2.0]])), k


@pytest.mark.parametrize("n", [1, 255, 300000])
def test_values_pack_to_the_nearest_step(n):
    r = np.random.RandomState(n)
    x = (r.standard_normal(n) * np.exp(r.standard_normal(n) * 3)).astype(np.float32).astype(np.float64)
    half = np.full(n, 0.5)
    m, v = packed(x, np.abs(x))
    assert np.array_equal(m, R.held(x, R.LEAST_M, half))
    assert np.array_equal(v, R.held(np.abs(x), R.LEAST_V, half, positive=True))


