"""CPU tests of the 8-bit moments' format as restated in numpy, and of the
argument checks that run before any GPU work."""
import numpy as np
import pytest
import torch

from cpuforge_amd import _lib
from tests import adamw8_ref as R


def test_mean_of_roundings_is_the_value():
    """A moment that moves by a thousandth of itself a step is followed: 4000
    steps' roundings average to it (their deviation: a step of at most an
    eighth, over sqrt(12 * 4000) in the mean of uniform thresholds)."""
    x = np.abs(np.random.RandomState(0).standard_normal(64)) + 0.1
    got = np.mean([R.held(x, R.LEAST_V, R.thresholds(x.size, t)[1], positive=True) for t in range(1, 4001)], axis=0)
    assert np.abs(got / x - 1).max() < 6 * 0.125 / 2 / np.sqrt(4000)


def test_a_held_state_is_held_as_it_is():
    r = np.random.RandomState(1)
    x = r.standard_normal(4096) * np.exp(r.standard_normal(4096) * 3)
    for least, pos in ((R.LEAST_M, False), (R.LEAST_V, True)):
        y = np.abs(x) if pos else x
        u = r.rand(x.size)
        once = R.held(y, least, u, pos)
        for again in (np.full(x.size, 0.5), r.rand(x.size)):
            assert np.array_equal(R.held(once, least, again, pos), once)
        live = np.abs(y) > np.exp2(R.exponent(R.blocks(np.abs(y))) + least).repeat(256, 1).reshape(-1)[:x.size]
        assert np.abs(once / y - 1)[live].max() <= 0.125


def test_thresholds_are_uniform_and_independent():
    a, b = R.thresholds(1 << 16, 7)
    a2, b2 = R.thresholds(1 << 16, 8)
    for x in (a, b):
        assert abs(x.mean() - 0.5) < 6 / np.sqrt(12 * x.size) and x.min() >= 0 and x.max() < 1
    for x, y in ((a, b), (a[1:], a[:-1]), (b[1:], b[:-1]), (a, a2), (b, b2)):
        assert abs(np.corrcoef(x, y)[0, 1]) < 6 / np.sqrt(x.size)


def test_state_bytes():
    L = _lib.lib()
    for n in (0, 1, 255, 256, 257, 4096, 10 ** 9):
        assert L.cfops_adamw8_state_bytes(n) == -(-n // 256) * 514


def test_null_contexts_are_refused():
    L = _lib.lib()
    assert L.cfops_lm_head_logprobs(None, None, None, None, 1, 1, 1, None, None, None, None, 0, None) == _lib.ERR_ARG
    assert L.cfops_lm_head_logprobs_backward(None, None, None, None, None, None, 1, 1, 1, None, None, 1, None, 0,
                                             None) == _lib.ERR_ARG
    assert L.cfops_preference_loss(None, None, None, None, 1, None, 1, 0, 0.1, 0.0, 0.0, 0, None, None, None,
                                   None) == _lib.ERR_ARG
    assert L.cfops_policy_loss(None, None, None, None, None, None, 1, None, 1, 0, 0.2, 0.2, 0.0, 0, None, None,
                               None) == _lib.ERR_ARG
    for f in (L.cfops_adamw8_pack_multi, L.cfops_adamw8_unpack_multi):
        assert f(None, 0, None, None) == _lib.ERR_ARG
    assert L.cfops_adamw8_update_multi(None, 0, None, 1, 0.1, 0.9, 0.9, 0.0, None) == _lib.ERR_ARG


def test_host_tensors_and_unknown_names_are_refused():
    from cpuforge_amd import ops as P
    x, i, r = torch.zeros(4), torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)
    off = torch.tensor([0, 2, 4])
    ctx = object()  # the checks come before its first use
    with pytest.raises(TypeError):
        P.lm_head_logprobs(x, x, i, 4, 1, 4, x, x, r, ctx=ctx)
    with pytest.raises(ValueError, match="form"):
        P.preference_loss(x, x, i, off, x, x[:2], r, beta=0.1, form="none", ctx=ctx)
    with pytest.raises(_lib.ShapeError):
        P.preference_loss(x, x, i, off[:2], x, x[:2], r, beta=0.1, ctx=ctx)
    with pytest.raises(TypeError):
        P.preference_loss(x, x, i, off, x, x[:2], r, beta=0.1, ctx=ctx)
    with pytest.raises(ValueError, match="reduction"):
        P.policy_loss(x, x, x, x, i, off, x, r, clip_low=0.2, clip_high=0.2, reduction="sum", ctx=ctx)
    with pytest.raises(TypeError):
        P.policy_loss(x, x, x, x, i, off, x, r, clip_low=0.2, clip_high=0.2, ctx=ctx)
    with pytest.raises(ValueError):
        P.Adamw8Tensors([dict(p=x, g=x)])
    with pytest.raises(TypeError):
        P.Adamw8Tensors([dict(p=x, g=x, m=x, v=x)])


def test_optimizer_state_bits():
    from cpuforge_amd.optim import AdamW
    with pytest.raises(ValueError):
        AdamW(0.9, 0.999, 1e-8, 0.0, state_bits=4)
