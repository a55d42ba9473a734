"""CPU tests of what ops.layernorm_*, rotary and lm_head_distill refuse before they
reach the library, and of the sizes that the library tells without a device."""
import pytest
import torch

from cpuforge_amd import ops as P


class Ctx:
    """A context that no call may reach."""
    device = 0


def test_host_tensors_are_refused():
    x, w, s = torch.zeros(4, 8), torch.zeros(8), torch.zeros(4)
    with pytest.raises(TypeError, match="device tensor"):
        P.layernorm_forward(x, w, w, x, s, s, 4, 8, 1e-5, ctx=Ctx())
    with pytest.raises(TypeError, match="device tensor"):
        P.layernorm_backward(x, x, w, s, s, x, w, w, 4, 8, ctx=Ctx())
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(TypeError, match="device tensor"):
        P.rotary(q, q, torch.zeros(4, 4), torch.zeros(4, 4), ctx=Ctx())
    with pytest.raises(TypeError, match="device tensor"):
        P.rotary([q, None], [q, q], torch.zeros(4, 4), torch.zeros(4, 4), ctx=Ctx())
    ids = torch.zeros(4, 3, dtype=torch.int64)
    with pytest.raises(TypeError, match="device tensor"):
        P.lm_head_distill(x, torch.zeros(9, 8), ids, ids.float(), 4, 8, 9, 3, s, torch.zeros(3, dtype=torch.int32),
                          ctx=Ctx())
    with pytest.raises(TypeError, match="device tensor"):
        P.lm_head_distill_backward(x, torch.zeros(9, 8), ids, ids.float(), s, 4, 8, 9, 3, ctx=Ctx())


def test_numbers_of_tensors():
    q = torch.zeros(1, 4, 2, 8)
    for xs, ys in (((), ()), ((q,) * 5, (q,) * 5), ((q, q), (q,))):
        with pytest.raises(ValueError, match="as many"):
            P.rotary(xs, ys, None, None, ctx=Ctx())


def test_keep_bytes():
    size = P.lm_head_distill_keep_bytes
    assert size(0, 64, 1000, 8) == size(100, 0, 1000, 8) == size(100, 64, 0, 8) == 0
    assert size(100, 64, 1000, 0) == size(100, 64, 1000, 1025) == size(1 << 24, 64, 1000, 8) == 0
    assert size(16, 64, 1000, 8) >= 16 * 1000 * 4 and size(24, 64, 1000, 8) >= 32 * 1000 * 4
    for k in (1, 8, 1024):  # what the products keep, and the entries
        assert size(100, 64, 1000, k) >= P.lm_head_logprobs_keep_bytes(100, 64, 1000) + 8 * 100 * k
