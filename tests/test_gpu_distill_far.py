"""GPU tests of cfops_lm_head_distill at the ends of its values' ranges, against the
definition in 64 bits, alike for few rows and for many."""
import math

import pytest
import torch

from cpuforge_amd import ops as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # half a step of f32


def forward(hn, head, ids, z, lse, keep=None):
    t, d = hn.shape
    loss, res = torch.full((t,), 77.0, device=DEV), P.ce_result_buffer(DEV)
    P.lm_head_distill(hn, head, ids, z, t, d, head.shape[0], ids.shape[1], loss, res, lse, 1.0, keep)
    return loss, res


def backward(hn, head, ids, z, lse, dloss, keep=None):
    dhn, dhead = torch.full_like(hn, 77.0), torch.full_like(head, 77.0)
    P.lm_head_distill_backward(hn, head, ids, z, dloss, *hn.shape, head.shape[0], ids.shape[1], dhn, dhead, lse, 1.0,
                               keep, acc=False)
    return dhn, dhead


def keep_of(hn, head, ids):
    n = P.lm_head_distill_keep_bytes(*hn.shape, head.shape[0], ids.shape[1])
    return torch.empty(n, dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("t", [20, 150])
def test_a_teacher_sum_of_minus_infinity_counts_as_the_entries_own(t):
    """It is below theirs, as any other that is (a cast of a value below f32's lowest)."""
    g = torch.Generator(device=DEV).manual_seed(t)
    hn, head = torch.randn(t, 48, generator=g, device=DEV), torch.randn(300, 48, generator=g, device=DEV) * 0.1
    ids = torch.rand(t, 300, generator=g, device=DEV).topk(6).indices
    z, dloss = torch.randn(t, 6, generator=g, device=DEV), torch.randn(t, generator=g, device=DEV)
    lowest = torch.full((t,), -math.inf, device=DEV)
    lowest[1] = torch.finfo(torch.float32).min
    out = []
    for lse in (None, lowest):
        keep = keep_of(hn, head, ids)
        loss, res = forward(hn, head, ids, z, lse, keep)
        P.distill_check(res)
        out.append((loss, *backward(hn, head, ids, z, lse, dloss, keep), *backward(hn, head, ids, z, lse, dloss)))
    for a, b in zip(*out):
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b)
