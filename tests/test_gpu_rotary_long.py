"""GPU tests of ops.rotary over more tokens than one launch takes, and of tensors that a
launch cannot take together."""
import pytest
import torch

from cpuforge_amd import ops as P
from cpuforge_amd._lib import CfattnError

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


def test_tensors_that_share_an_output_are_refused():
    """One launch turns all tensors: a y that is another's, or another's x, would have either."""
    cos, sin = torch.zeros(5, 4, device=DEV), torch.ones(5, 4, device=DEV)
    a, b, c, d = (torch.randn(1, 5, 2, 8, device=DEV) for _ in range(4))
    was = [t.clone() for t in (a, b, c, d)]
    for xs, ys in (((a, b), (c, c)), ((a, b), (b, c)), ((a, b), (c, a)), ((a, a), (a, a)), ((a, b, c), (d, b, d))):
        with pytest.raises(CfattnError, match="share"):
            P.rotary(xs, ys, cos, sin)
    assert all(torch.equal(t, w) for t, w in zip((a, b, c, d), was))
    P.rotary((a, a), (c, d), cos, sin)  # (two outputs of one input are two)
    assert torch.equal(c, d)
