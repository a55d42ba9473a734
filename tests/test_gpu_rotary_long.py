"""GPU test of ops.rotary over more tokens than one launch takes."""
import pytest
import torch

from cpuforge_amd import ops as P

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("heads", [(3,), (3, 5)])
def test_each_token_is_turned_once(heads):
    """In place, over 2^23 / (tensors) tokens to a launch, which 85 (51) tokens to a
    workgroup do not divide: the workgroup at a launch's end has room for tokens of the next.
    By a quarter turn, so that every value is exact: (a, b) -> (-b, a)."""
    tokens = (1 << 23) + 1000
    cos, sin = torch.zeros(tokens, 1, device=DEV), torch.ones(tokens, 1, device=DEV)
    xs = [torch.randn(1, tokens, h, 2, device=DEV) for h in heads]
    want = [torch.stack([-x[..., 1], x[..., 0]], -1) for x in xs]
    ys = [torch.empty_like(x) for x in xs]
    P.rotary(xs, ys, cos, sin)
    P.rotary(xs, xs, cos, sin)
    for x, y, w in zip(xs, ys, want):
        assert torch.equal(y, w)
        wrong = torch.nonzero((x != w).flatten(2).any(-1))
        assert not len(wrong), wrong[:8].tolist()
