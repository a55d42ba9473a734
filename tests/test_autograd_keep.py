"""CPU tests of when autograd.lm_head_logprobs has its forward keep what a
backward reads: the library's call is replaced by one that notes its keep."""
import pytest
import torch

from cpuforge_amd import autograd as A
from cpuforge_amd import ops as P


@pytest.fixture
def keeps(monkeypatch):
    seen = []

    def forward(hn, head, targets, t, d, vocab, logp, lse, result, keep=None, ctx=None):
        seen.append(None if keep is None else keep.numel())
        logp.zero_()

    monkeypatch.setattr(P, "lm_head_logprobs", forward)
    monkeypatch.setattr(P, "lm_head_logprobs_keep_bytes", lambda t, d, vocab: 4 * t * vocab)
    return seen


def call(hn_grad, head_grad):
    hn, head = torch.zeros(5, 3, requires_grad=hn_grad), torch.nn.Parameter(torch.zeros(7, 3), requires_grad=head_grad)
    return A.lm_head_logprobs(hn, head, torch.zeros(5, dtype=torch.int64))


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("hn_grad,head_grad", [(False, True), (True, False), (True, True), (False, False)])
def test_nothing_is_kept_where_no_backward_can_follow(keeps, mode, hn_grad, head_grad):
    with mode():
        logp, _ = call(hn_grad and mode is torch.no_grad, head_grad)
    assert keeps == [None] and not logp.requires_grad


@pytest.mark.parametrize("hn_grad,head_grad", [(False, True), (True, False), (True, True)])
def test_a_forward_keeps_for_its_backward(keeps, hn_grad, head_grad):
    logp, block = call(hn_grad, head_grad)
    assert keeps == [4 * 5 * 7] and logp.requires_grad and not block.requires_grad


def test_frozen_operands_keep_nothing(keeps):
    logp, _ = call(False, False)
    assert keeps == [None] and not logp.requires_grad


def test_the_limit_holds(keeps, monkeypatch):
    monkeypatch.setattr(A, "LOGPROBS_KEEP_LIMIT", 4 * 5 * 7 - 1)
    assert call(True, True)[0].requires_grad and keeps == [None]


@pytest.mark.gpu
def test_a_trainable_head_without_a_gradient_takes_a_frozen_ones_memory():
    """The peak of a call under no_grad on the device, by the library's own call."""
    def peak(head_grad):
        hn = torch.randn(300, 64, device="cuda")
        head = torch.nn.Parameter(torch.randn(20000, 64, device="cuda"), requires_grad=head_grad)
        tg = torch.arange(300, device="cuda")
        with torch.no_grad():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            logp, _ = A.lm_head_logprobs(hn, head, tg)
            torch.cuda.synchronize()
            return torch.cuda.max_memory_allocated() - before, logp
    (frozen, want), (trains, got) = peak(False), peak(True)
    assert trains == frozen and want.shape == got.shape
