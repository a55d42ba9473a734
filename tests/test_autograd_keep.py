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


def test_the_function_itself_takes_three_arguments(keeps, monkeypatch):
    monkeypatch.setattr(P, "lm_head_logprobs_backward", lambda hn, head, *a, acc: (a[6].fill_(1.0), a[7].fill_(2.0)))
    hn, head = torch.zeros(5, 3, requires_grad=True), torch.zeros(7, 3, requires_grad=True)
    logp, _ = A.LMHeadLogprobsFn.apply(hn, head, torch.zeros(5, dtype=torch.int64))
    logp.sum().backward()
    assert keeps == [4 * 5 * 7] and bool((hn.grad == 1.0).all()) and bool((head.grad == 2.0).all())


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


@pytest.mark.gpu
@pytest.mark.parametrize("rows,keeps", [((4, 15), False), ((4, 35), True), ((2, 5, 70), True)])
def test_gradients_are_those_of_the_calls_with_what_the_forward_keeps(rows, keeps):
    """Bit for bit, of hidden states and head together and of either alone; and they
    are the 64-bit gradients to f32 products (2^-20 of the largest)."""
    t, d, vocab = torch.Size(rows).numel(), 48, 500
    gen = torch.Generator(device="cuda").manual_seed(t)
    hn = torch.randn(*rows, d, generator=gen, device="cuda").requires_grad_()
    head = (torch.randn(vocab, d, generator=gen, device="cuda") * 0.3).requires_grad_()
    tg = torch.randint(0, vocab, rows, generator=gen, device="cuda")
    tg.view(-1)[::5] = P.IGNORE_INDEX
    g = torch.randn(*rows, generator=gen, device="cuda")

    n = P.lm_head_logprobs_keep_bytes(t, d, vocab)
    assert (n > 0) == keeps
    keep = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
    logp, lse = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
    flat = (hn.detach().view(t, d), head.detach(), tg.view(-1))
    P.lm_head_logprobs(*flat, t, d, vocab, logp, lse, P.ce_result_buffer("cuda"), keep)
    dhn, dhead = torch.empty(t, d, device="cuda"), torch.empty(vocab, d, device="cuda")
    P.lm_head_logprobs_backward(*flat, lse, g.view(-1), t, d, vocab, dhn, dhead, keep, acc=False)

    got, _ = A.lm_head_logprobs(hn, head, tg)
    assert got.shape == tg.shape and torch.equal(got.view(-1), logp)
    both = torch.autograd.grad(got, (hn, head), g)
    assert torch.equal(both[0].view(t, d), dhn) and torch.equal(both[1], dhead)
    (one,) = torch.autograd.grad(A.lm_head_logprobs(hn, head.detach(), tg)[0], hn, g)
    (other,) = torch.autograd.grad(A.lm_head_logprobs(hn.detach(), head, tg)[0], head, g)
    assert torch.equal(one, both[0]) and torch.equal(other, both[1])

    h, w = hn.detach().double().view(t, d), head.detach().double()
    hot = torch.zeros(t, vocab, dtype=torch.float64, device="cuda").scatter_(1, tg.view(-1, 1).clamp(min=0), 1.0)
    D = (hot - torch.softmax(h @ w.T, 1)) * ((tg != P.IGNORE_INDEX) * g).double().view(t, 1)
    for x, want in ((dhn, D @ w), (dhead, D.T @ h)):
        assert bool(((x.double() - want).abs() <= 2.0 ** -20 * want.abs().max()).all())
