"""GPU tests of cfops_lm_head_logprobs_backward where tokens are nearly certain and
logits large: every logit is exact in f32, so the probabilities' error is theirs
alone, whatever the size of lse."""
import pytest
import torch

from tests.test_gpu_head_grad import DEV, FORMS, IGN, U, gradients, report

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,keeps", FORMS + [(1, False), (20, False)])
def test_gradients_of_likely_tokens_beside_large_logits(t, keeps):
    """Logits of 4096 and some: a target's lies some 6 above the others, 1 - P about
    1e-2; 4096 is common to all of them, which no gradient sees."""
    vocab, d = 1500, 32
    gen = torch.Generator(device=DEV).manual_seed(t)
    head = torch.randint(-2, 3, (vocab, d), generator=gen, device=DEV) * 0.5
    tg = torch.randint(0, vocab, (t,), generator=gen, device=DEV)
    hn = head[tg].contiguous()
    head[:, 0], hn[:, 0] = 64.0, 64.0
    g = torch.randn(t, generator=gen, device=DEV)
    tg[3:4] = IGN
    use = (tg != IGN)[:, None]
    h, w = hn.double(), head.double()
    x = h @ w.T
    assert torch.equal(x, x.float().double()) and float(x.max()) > 4096
    P = torch.softmax(x, 1) * use
    hot = torch.zeros_like(P).scatter_(1, tg.clamp(min=0)[:, None], 1.0) * use
    ag = g.abs().double()[:, None]
    dx = (hot - P) * g.double()[:, None]
    # A probability: some 64 roundings (its argument's, 2^-24 of a difference of 30, exp's,
    # the sum's); 1 - P at the target: P's own beside it.
    off = ag * U * (64 * P + 4 * hot)
    dhn, dhead = gradients(hn, head, tg, g, keeps)
    want = dx @ w
    bound = off @ w.abs() + U * (vocab / 64 + 32) * ((ag * (P + hot)) @ w.abs()) + 2.0 ** -126
    report("dhn", (dhn - want).abs(), bound, want[:, 1:])
    assert bool(((dhn - want).abs() <= bound).all())
    want = dx.T @ h
    bound = off.T @ h.abs() + U * (t / 16 + 16) * (dx.abs().T @ h.abs()) + U * want.abs() \
        + 2.0 ** -38 * t * (dx.abs() * h.abs().amax(1, keepdim=True)).amax(0)[:, None] + 2.0 ** -126
    report("dhead", (dhead - want).abs(), bound, want)
    assert bool(((dhead - want).abs() <= bound).all())
