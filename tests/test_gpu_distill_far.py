"""GPU tests of cfops_lm_head_distill at the ends of its values' ranges, against the
definition in 64 bits, alike for few rows and for many."""
import math
import random

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


class Exact:
    """The loss and the gradients of 1 as temperature, the rest's in logarithms: q_v p_rest /
    q_rest is p_rest exp(log q_v - log q_rest), whatever q_rest is.  What they may be off: the
    logits by the rounding of 22-bit operands and f32 sums (`off`); logarithms by 2^-24 of the
    exponents that they join (the factor from logits to powers of two is an f32) and of some 40
    values; the rest by 2^-18 for each entry beside which it is summed; a gradient by 2^-36 of
    its part's and what sums over its terms round."""

    def __init__(self, hn, head, ids, z, lse, dloss):
        h, w, g = hn.double(), head.double(), dloss.double()[:, None]
        x = h @ w.T
        log_q = torch.log_softmax(x, 1)
        named = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids, True)
        p = torch.zeros_like(x).scatter_(1, ids, (z.double() - lse.double()[:, None]).exp())
        p_rest = -torch.expm1(z.double().logsumexp(1) - lse.double())
        log_rest = log_q.masked_fill(named, -math.inf).logsumexp(1)
        self.loss = (torch.xlogy(p, p) - p * log_q).where(named, torch.zeros(())).sum(1) \
            + p_rest * (p_rest.log() - log_rest)
        part = torch.where(named, 0.0, p_rest[:, None] * (log_q - log_rest[:, None]).exp())
        q = log_q.exp()
        dx = torch.where(named, q - p, q - part) * g
        self.dhn, self.dhead = dx @ w, dx.T @ h
        n, vocab, t = ids.shape[1], head.shape[0], hn.shape[0]
        off = (2.0 ** -22 + 2 * U) * (h.abs() @ w.abs().T).amax(1)
        spread = x.amax(1) - x.amin(1)
        tol = off + U * (vocab / 512 + 40 + spread)
        rest = off + tol + n * 2.0 ** -18
        self.tol_loss = off + tol + p_rest * rest + U * self.loss.abs()
        rel = (off + tol + U * (spread + 8))[:, None]
        e = q * rel + part * rest[:, None] + 2.0 ** -36
        e = e * g.abs() + dx.abs() * (2.0 ** -21 + U * vocab ** 0.5 + U * n)
        self.tol_dhn = e @ w.abs()
        self.tol_dhead = e.T @ h.abs() + U * self.dhead.abs() + U * t ** 0.5 * (dx.abs().T @ h.abs())
        # How much of dhn is the rest's: what a test of it has to tell from nothing.
        self.of_rest = (part * g.abs()) @ w.abs()


class Drawn(Exact):
    """The same where logits are sums of terms of any size, and parts of the rest of any below
    their entry: the three products of 16 k each round an f32 sum, 2^-24 of the largest each, and
    an exponential is taken to 2^-36 of its part's largest, 2^-33 where the rows of the head
    beside it are up to 8 times smaller, times the factor of the rest (2^10 at most of a part that
    is not scaled up)."""

    def __init__(self, hn, head, ids, z, lse, dloss):
        super().__init__(hn, head, ids, z, lse, dloss)
        h, w, g = hn.double(), head.double(), dloss.double()[:, None].abs()
        x = h @ w.T
        log_q = torch.log_softmax(x, 1)
        named = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids, True)
        p_rest = -torch.expm1(z.double().logsumexp(1) - lse.double())
        log_rest = log_q.masked_fill(named, -math.inf).logsumexp(1)
        part = torch.where(named, 0.0, p_rest[:, None] * (log_q - log_rest[:, None]).exp())
        more = 2 * 3 * math.ceil(h.shape[1] / 16) * U * (h.abs() @ w.abs().T).amax(1)
        steep = (p_rest.log() - log_rest).clamp(max=10 * math.log(2.0)).exp()
        e = ((log_q.exp() + part) * more[:, None] + 2.0 ** -33 * (1 + steep[:, None])) * g
        self.tol_loss = self.tol_loss + (1 + p_rest) * more
        self.tol_dhn = self.tol_dhn + e @ w.abs()
        self.tol_dhead = self.tol_dhead + e.T @ h.abs()


def check(hn, head, ids, z, lse, dloss, exact=Exact):
    w = exact(hn, head, ids, z, lse, dloss)
    keep = keep_of(hn, head, ids)
    loss, res = forward(hn, head, ids, z, lse, keep)
    P.distill_check(res)
    assert math.isfinite(float(P.ce_result_loss(res)))
    for k in (keep, None):
        dhn, dhead = backward(hn, head, ids, z, lse, dloss, k)
        for got, want, tol in ((loss, w.loss, w.tol_loss), (dhn, w.dhn, w.tol_dhn), (dhead, w.dhead, w.tol_dhead)):
            off = (got.double() - want).abs()
            assert bool((off <= tol).all()), (float((off - tol).max()), float(off.max()))
    if exact is Drawn:
        return
    assert bool(((w.tol_dhn < 0.1 * w.of_rest).sum(1) > hn.shape[1] / 2).all())


@pytest.mark.parametrize("gap", [45.0, 60.0, 100.0, 300.0])
@pytest.mark.parametrize("t", [20, 150])
def test_what_sums_of_entries_round_is_no_rest(t, gap):
    """Several entries of a like size in one part of the vocabulary, others 16 below them in
    another and 28 below in a third, and the rest `gap` below: what is left of an f32 sum
    less its entries is their rounding, 2^-24 of the largest, and far above the rest.  Parts
    of the rest alone, one of them far below another, and none."""
    g = torch.Generator(device=DEV).manual_seed(t)
    d, k = 64, 14
    dloss = torch.randn(t, generator=g, device=DEV)
    for vocab in (900, 380):
        hn, head = torch.randn(t, d, generator=g, device=DEV), torch.randn(vocab, d, generator=g, device=DEV) * 0.05
        ids = torch.tensor([3, 20, 50, 90, 101, 127, 130, 150, 199, 201, 240, 256, 300, 379], device=DEV)
        z = torch.randn(t, k, generator=g, device=DEV)
        lse = (z.double().logsumexp(1) - math.log1p(-0.2)).float()
        hn[:, 0], head[:, 0], head[500:, 0] = 8.0, 0.0, -2.0
        head[ids[:6], 0], head[ids[6:11], 0], head[ids[11:], 0] = gap / 8, (gap - 16) / 8, (gap - 28) / 8
        check(hn, head, ids.expand(t, k).contiguous(), z, lse, dloss)


@pytest.mark.parametrize("gap", [600.0, 690.0, 720.0, 1000.0, 4000.0])
@pytest.mark.parametrize("t", [20, 150])
def test_a_rest_that_64_bits_do_not_hold(t, gap):
    """Every entry is `gap` above every other token, two of them in one part of the
    vocabulary and one in another: the rest is e^-gap and less, and has its share of the loss
    and all of its gradient, however many rows there are.  With two parts of the rest
    alone, one of which is far below the other, and with entries in each part."""
    g = torch.Generator(device=DEV).manual_seed(t)
    dloss = torch.randn(t, generator=g, device=DEV)
    for vocab, entries in ((700, [5, 9, 140]), (300, [5, 140, 141, 260, 299])):
        d, k = 64, len(entries)
        hn, head = torch.randn(t, d, generator=g, device=DEV), torch.randn(vocab, d, generator=g, device=DEV) * 0.05
        ids = torch.tensor(entries, device=DEV).expand(t, k).contiguous()
        z = torch.randn(t, k, generator=g, device=DEV)
        lse = (z.double().logsumexp(1) - math.log1p(-0.2)).float()
        hn[:, 0], head[:, 0] = gap / 4, 0.0
        head[400:, 0] = -0.25
        head[entries, 0] = 4.0
        check(hn, head, ids, z, lse, dloss)


@pytest.mark.parametrize("below", [30.0, 59.0, 70.0, 90.0, 200.0])
def test_values_just_below_a_power_of_two(below):
    """A part of the vocabulary whose entry is 2^`below` above its largest other token, which is
    scaled up for the gradient's product, to all but 2^-13 of a power of two; it stands among
    rows of the head that are 8 times as large as those before them, which the product takes
    with a scale of their own: the scaled value has to be within what f16 holds."""
    t, d, vocab = 150, 32, 300
    g = torch.Generator(device=DEV).manual_seed(7)
    hn, head = torch.zeros(t, d, device=DEV), torch.rand(vocab, d, generator=g, device=DEV) * 2 - 1
    head[:, 31] = 1.0  # (the power of two of each 32 rows)
    head[32:64] *= 8.0
    hn[:, 0], hn[:, 1] = 256.0, torch.arange(t, device=DEV) % 4  # (rows are alike but for a little)
    unit = math.log(2.0) / 256
    head[:, 0], head[:, 1] = -(below + 5) * unit, 0.0
    head[40, 0], head[40, 1] = -(below + 0.00017) * unit, 0.00002 * 256 * unit
    head[3, 0] = 0.0
    ids = torch.full((t, 1), 3, device=DEV)
    z = torch.zeros(t, 1, device=DEV)
    lse = torch.full((t,), -math.log1p(-0.2), device=DEV)
    check(hn, head, ids, z, lse, torch.randn(t, generator=g, device=DEV))


@pytest.mark.parametrize("low", [-104.5, -106.0, -108.0])
def test_tokens_whose_probabilities_f32_does_not_hold(low):
    """Tokens of 2^-151 of the largest and less in a part whose largest is 2^-144, beside a rest
    of 2^-58 whose gradient is 2^55 times as steep: probability times factor is in f32 what
    the probability alone is not, and the head's gradient takes its scale from the product."""
    t, d, vocab = 150, 64, 384
    g = torch.Generator(device=DEV).manual_seed(3)
    hn, head = torch.randn(t, d, generator=g, device=DEV), torch.randn(vocab, d, generator=g, device=DEV) * 0.01
    hn[:, 0], head[:, 0] = 8.0, low / 8
    head[:256, 0], head[256, 0] = -45.0 / 8, -100.0 / 8
    head[[3, 20], 0] = 0.0
    ids = torch.tensor([3, 20], device=DEV).expand(t, 2).contiguous()
    z = torch.randn(t, 2, generator=g, device=DEV)
    lse = (z.double().logsumexp(1) - math.log1p(-0.2)).float()
    check(hn, head, ids, z, lse, torch.randn(t, generator=g, device=DEV))


@pytest.mark.parametrize("seed", range(60))
def test_drawn_students(seed):
    """Entries and others at levels up to 500 apart, in parts of any mixture, over rows of the
    head of one size or of many, with gradients of any size."""
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, d, vocab = rng.choice((20, 64, 65, 150, 300)), rng.choice((16, 33, 64, 200)), rng.choice((130, 300, 700, 5000))
    k = rng.choice((1, 2, 5, 12, 40, 100))
    levels = torch.tensor([rng.choice((0.0, 5.0, rng.uniform(0, 60), rng.uniform(30, 160), 500.0)) for _ in range(3)])
    hn = torch.randn(t, d, generator=g, device=DEV)
    head = torch.randn(vocab, d, generator=g, device=DEV) * rng.choice((0.05, 0.3, 1.0)) * 4 / d ** 0.5
    ids = torch.randperm(vocab, generator=g, device=DEV)[:k]
    if seed % 2:
        ids = torch.arange(k, device=DEV) + rng.randrange(vocab - k)
    hn[:, 0], head[:, 0] = 8.0, 0.0
    head[ids, 0] = levels.to(DEV)[torch.randint(0, 3, (k,), generator=g, device=DEV)] / 8
    if seed % 3 == 0:
        head[torch.randperm(vocab, generator=g, device=DEV)[:vocab // 3], 0] -= rng.uniform(0, 20)
    if seed % 4 == 0:
        head[:, 1:] *= torch.exp(2 * torch.randn(vocab, 1, generator=g, device=DEV))
    z = torch.randn(t, k, generator=g, device=DEV) * rng.choice((0.3, 1.0, 5.0))
    share = rng.choice((1e-5, 0.01, 0.2, 0.9, 0.9999))
    lse = (z.double().logsumexp(1) - math.log1p(-share)).float()
    dloss = torch.randn(t, generator=g, device=DEV) * 10.0 ** rng.choice((0, 0, -15, 12))
    check(hn, head, ids.expand(t, k).contiguous(), z, lse, dloss, Drawn)
