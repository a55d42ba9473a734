"""GPU tests of distillation from a teacher's top logits through the LM head
(cfops_lm_head_distill, _backward) against the definition in 64 bits."""
import math

import pytest
import torch

from cpuforge_amd import autograd as A
from cpuforge_amd import ops as P
from cpuforge_amd._lib import CfattnError, ShapeError

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = P.IGNORE_INDEX
U = 2.0 ** -24  # half a step of f32
NONE = 2 ** 31 - 1


def inputs(t, d, vocab, k, seed, sharp=1.0, ragged=True, masked=0.2):
    """A student whose logits follow the teacher's by `sharp`."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)
    head = rand(vocab, d) / d ** 0.5
    k_have = min(k, vocab)
    ids = torch.rand(t, vocab, generator=g, device=DEV).topk(k_have, 1).indices
    z = 6 - 2 * torch.log1p(torch.arange(k_have, device=DEV).float()) + 0.5 * rand(t, k_have)
    hn = rand(t, d) + sharp * (z[:, :, None] * head[ids]).sum(1) / (head * head).sum(1).mean()
    if k > k_have:  # entries that are not there
        ids = torch.cat([ids, torch.full((t, k - k_have), IGN, device=DEV)], 1)
        z = torch.cat([z, rand(t, k - k_have)], 1)
    if ragged:
        n = torch.randint(1, k + 1, (t, 1), generator=g, device=DEV)
        gone = torch.rand(t, k, generator=g, device=DEV).argsort(1) >= n
        half = torch.rand(t, k, generator=g, device=DEV) < 0.5
        ids = torch.where(gone & half, IGN, ids)
        z = torch.where(gone & ~half, -math.inf, z)
    ids[torch.rand(t, generator=g, device=DEV) < masked] = IGN
    return hn, head, ids.contiguous(), z.contiguous(), rand(t)


def teacher_lse(ids, z, temp, share=0.1):
    own = torch.where(ids == IGN, -math.inf, z.double() / temp).logsumexp(1)
    return torch.nan_to_num(own - math.log1p(-share), neginf=0.0).float()


class Exact:
    """The loss and its gradients, and how far a product of 22-bit operands in f32
    sums may be off (the logits by `off`, as the log-probabilities' tests count
    them, and by a rounding of hn over the temperature)."""

    def __init__(self, hn, head, ids, z, lse, temp, dloss):
        t, vocab = hn.shape[0], head.shape[0]
        h, w = hn.double() / temp, head.double()
        x = h @ w.T
        there = (ids != IGN) & (z != -math.inf)
        self.use = there.any(1)
        zt = torch.where(there, z.double() / temp, -math.inf)
        own = zt.logsumexp(1)
        whole = own if lse is None else torch.maximum(own, lse.double())
        p = torch.zeros(t, vocab, dtype=torch.float64, device=DEV)
        named = torch.zeros(t, vocab, dtype=torch.bool, device=DEV)
        r, c = torch.nonzero(there, as_tuple=True)
        named[r, ids[r, c]] = True
        every = named.all(1)
        whole = torch.where(every, own, whole)
        p[r, ids[r, c]] = (zt - whole[:, None])[r, c].exp()
        log_q = torch.log_softmax(x, 1)
        q = log_q.exp()
        p_rest = -torch.expm1(own - whole) if lse is not None else torch.zeros_like(own)
        p_rest = torch.where(self.use, p_rest, 0.0)
        log_rest = log_q.masked_fill(named, -math.inf).logsumexp(1)
        some = p_rest > 0
        ratio = torch.where(some, p_rest / log_rest.exp(), 0.0)
        loss = torch.where(named, torch.xlogy(p, p) - p * log_q, 0.0).sum(1)
        rest = p_rest * (p_rest.clamp(min=1e-300).log() - torch.where(some, log_rest, 0.0))
        loss = loss + torch.where(some, rest, 0.0)
        dx = torch.where(named, q - p, q * (1 - ratio)[:, None])
        g = torch.where(self.use, dloss.double(), 0.0)
        self.loss = torch.where(self.use, loss, 0.0)
        self.dx = torch.where(self.use[:, None], dx * g[:, None], 0.0)
        self.dhn, self.dhead = self.dx @ w / temp, self.dx.T @ h
        # Errors.
        n = there.sum(1).double()
        off = (2.0 ** -22 + 2 * U) * (h.abs() @ w.abs().T).amax(1)
        spread = (x.amax(1) - x.amin(1)).clamp(max=104.0)
        tol = off + U * (vocab / 512 + 40 + spread)  # of the logarithm of the sum
        # A rest may be what the sums of 128 leave, each to 2^-18 of the rest.
        rest = off + tol + n * 2.0 ** -18
        self.tol_loss = torch.where(self.use, off + tol + p_rest * rest + U * loss.abs(), 0.0)
        rel = (off + tol + U * (spread + 8))[:, None]
        e = torch.where(named, q * rel, q * ((1 - ratio).abs()[:, None] * rel + (ratio * rest)[:, None]))
        e = (e + dx.abs() * (2.0 ** -21 + U * vocab ** 0.5 + U * n[:, None]) + 2.0 ** -36) * g.abs()[:, None]
        e = torch.where(self.use[:, None], e, 0.0)
        self.tol_dhn = e @ w.abs() / temp + 1e-37
        self.tol_dhead = e.T @ h.abs() + U * (1 + self.dhead.abs()) \
            + U * t ** 0.5 * (self.dx.abs().T @ h.abs()) + 1e-37


def forward(hn, head, ids, z, lse, temp, keep=None):
    t, d = hn.shape
    loss, res = torch.full((t + 3,), 77.0, device=DEV), P.ce_result_buffer(DEV)
    P.lm_head_distill(hn, head, ids, z, t, d, head.shape[0], ids.shape[1], loss[:t], res, lse, temp, keep)
    assert bool((loss[t:] == 77.0).all())
    return loss[:t], res


def kept(hn, head, ids, z, lse, temp):
    n = P.lm_head_distill_keep_bytes(*hn.shape, head.shape[0], ids.shape[1])
    keep = torch.full((n + 64,), 255, dtype=torch.uint8, device=DEV)
    loss, _ = forward(hn, head, ids, z, lse, temp, keep[:n])
    assert bool((keep[n:] == 255).all())
    return keep[:n], loss


def backward(hn, head, ids, z, lse, temp, dloss, keep=None, acc=False, want_head=True):
    dhn = torch.full_like(hn, 77.0)
    dhead = torch.ones_like(head) if want_head else None
    P.lm_head_distill_backward(hn, head, ids, z, dloss, *hn.shape, head.shape[0], ids.shape[1], dhn, dhead, lse, temp,
                               keep, acc=acc)
    return dhn, dhead


def near(got, want, tol, what):
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (what, float((off - tol).max()), float(off.max()))


def check(hn, head, ids, z, lse, temp, dloss):
    w = Exact(hn, head, ids, z, lse, temp, dloss)
    loss, res = forward(hn, head, ids, z, lse, temp)
    P.distill_check(res)
    near(loss, w.loss, w.tol_loss, "loss")
    n = int(w.use.sum())
    assert int(res[0]) == n
    mean = float(w.loss.sum()) / max(n, 1)
    assert abs(float(P.ce_result_loss(res)) - mean) <= float(w.tol_loss.max()) + 2 * U * abs(mean)
    k = kept(hn, head, ids, z, lse, temp)
    assert torch.equal(k[1], loss)  # (the same products, whether or not they are kept)
    for keep in (None, k[0]):
        dhn, dhead = backward(hn, head, ids, z, lse, temp, dloss, keep)
        near(dhn, w.dhn, w.tol_dhn, "dhn")
        assert not dhn[~w.use].any()
        near(dhead, w.dhead, w.tol_dhead, "dhead")
        only, _ = backward(hn, head, ids, z, lse, temp, dloss, keep, want_head=False)
        assert torch.equal(only, dhn)
        _, added = backward(hn, head, ids, z, lse, temp, dloss, keep, acc=True)
        near(added, w.dhead + 1, w.tol_dhead, "dhead +")
    return loss


SHAPES = [(1, 1, 2, 1), (1, 64, 5, 5), (3, 7, 130, 4), (1, 576, 4097, 32), (16, 100, 1000, 64), (17, 576, 1000, 8),
          (33, 40, 128, 65), (64, 33, 4099, 20), (65, 31, 257, 33), (66, 2100, 300, 3), (70, 1500, 300, 300),
          (130, 100, 257, 130), (256, 64, 512, 64), (300, 65, 50, 70), (513, 576, 8192, 64), (700, 128, 900, 200),
          (90, 16, 5000, 1024), (5, 16, 5000, 1024), (1000, 16, 20000, 1),
          # More parts and slices of the vocabulary than a wave has at once.
          (70, 16, 140000, 8), (3, 8, 270000, 5)]


@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("t,d,vocab,k", SHAPES)
def test_shapes(t, d, vocab, k, rest):
    temp = (1.0, 2.0, 0.7)[(t + k) % 3]
    hn, head, ids, z, dloss = inputs(t, d, vocab, k, t + k, ragged=k > 1)
    check(hn, head, ids, z, teacher_lse(ids, z, temp) if rest else None, temp, dloss)


@pytest.mark.parametrize("share", [1e-4, 0.3])
@pytest.mark.parametrize("sharp", [0.0, 2.0, 4.0])
@pytest.mark.parametrize("t", [40, 200])
def test_students_from_uniform_to_sure(t, sharp, share):
    """What a sure student leaves to the rest is a sum of its own, not 1 less the others."""
    hn, head, ids, z, dloss = inputs(t, 300, 1500, 20, 7, sharp=sharp)
    check(hn, head, ids, z, teacher_lse(ids, z, 1.0, share=share), 1.0, dloss)
    check(hn, head, ids, z, None, 1.0, dloss)


@pytest.mark.parametrize("t", [20, 150])
def test_a_rest_far_below_the_entries(t):
    """One token of each row holds all but e^-40 of the student's probability, so every
    rest is formed from exponentials far below 2^-24 of the sums they stand in; at e^-120
    and below from logits formed again, where f32 holds no exponential and no p_rest / q_rest."""
    g = torch.Generator(device=DEV).manual_seed(t)
    d, vocab = 64, 700
    head = torch.randn(vocab, d, generator=g, device=DEV) * 0.05
    ids = torch.randint(0, vocab, (t, 1), generator=g, device=DEV)
    ids = torch.cat([ids, (ids + 1) % vocab], 1).contiguous()
    z = torch.randn(t, 2, generator=g, device=DEV)
    hn = torch.randn(t, d, generator=g, device=DEV)
    dloss = torch.randn(t, generator=g, device=DEV)
    lse = teacher_lse(ids, z, 1.0, share=0.2)
    own = head[ids[:, 0]]
    for far in (40.0, 60.0, 120.0, 400.0):
        check(hn + far / (own * own).sum(1, keepdim=True) * own, head, ids, z, lse, 1.0, dloss)


@pytest.mark.parametrize("t", [20, 150])
def test_a_rest_far_below_entries_in_every_part(t):
    """As above with entries in each 128 tokens, some far above, some among the others: no
    part of the vocabulary is of the rest alone."""
    g = torch.Generator(device=DEV).manual_seed(t)
    d, vocab = 64, 300
    head = torch.randn(vocab, d, generator=g, device=DEV) * 0.05
    ids = (torch.tensor([5, 100, 130, 200, 290], device=DEV) + torch.arange(t, device=DEV)[:, None] % 5).contiguous()
    z = torch.randn(t, 5, generator=g, device=DEV)
    hn = torch.randn(t, d, generator=g, device=DEV)
    dloss = torch.randn(t, generator=g, device=DEV)
    head[[5, 6, 7, 8, 9, 130, 131, 132, 133, 134], 0] = 3.0
    for far in (30.0, 90.0, 200.0):
        hn[:, 0] = far
        head[head[:, 0] != 3.0, 0] = 0.0
        check(hn, head, ids, z, teacher_lse(ids, z, 1.0, share=0.2), 1.0, dloss)


@pytest.mark.parametrize("t", [30, 300])
def test_entries_that_the_student_holds_for_impossible(t):
    """Entries 150 below the largest logit of their 128 tokens, whose exponentials f32 does
    not hold: their logits are formed again."""
    hn, head, ids, z, dloss = inputs(t, 96, 600, 12, 3, sharp=0.0)
    hn[:, 0] = 15.0
    head[:, 0] = 0.0
    head[5::128, 0] = 10.0  # the largest of each 128
    ids = torch.where(ids % 128 == 5, IGN, ids)
    check(hn, head, ids, z, teacher_lse(ids, z, 1.0, share=0.2), 1.0, dloss)


@pytest.mark.parametrize("t", [30, 100])
def test_every_token_is_an_entry(t):
    """There is no rest then, whatever the teacher's log-sum-exp."""
    hn, head, ids, z, dloss = inputs(t, 32, 40, 40, 5, ragged=False)
    a = check(hn, head, ids, z, None, 1.0, dloss)
    b = check(hn, head, ids, z, teacher_lse(ids, z, 1.0, share=0.3), 1.0, dloss)
    assert torch.equal(a, b)


@pytest.mark.parametrize("t", [50, 200])
def test_a_teacher_sum_below_the_entries_counts_as_theirs(t):
    hn, head, ids, z, dloss = inputs(t, 48, 500, 10, 5)
    lse = teacher_lse(ids, z, 1.0) - 5.0
    a = check(hn, head, ids, z, lse, 1.0, dloss)
    b, _ = forward(hn, head, ids, z, None, 1.0)
    assert torch.equal(a, b)


@pytest.mark.parametrize("t", [20, 150])
def test_order_of_entries_changes_no_bit(t):
    hn, head, ids, z, dloss = inputs(t, 64, 900, 40, 5)
    lse = teacher_lse(ids, z, 2.0)
    perm = torch.randperm(40, device=DEV)
    a, b = ((ids, z), (ids[:, perm].contiguous(), z[:, perm].contiguous()))
    # (Sums of the entries' exponentials in 64 bits are in their order: the last bit of an f32
    # loss may follow, no more.)
    la, lb = forward(hn, head, *a, lse, 2.0)[0], forward(hn, head, *b, lse, 2.0)[0]
    assert bool(((la - lb).abs() <= 2 * U * la.abs()).all())
    ga, gb = backward(hn, head, *a, lse, 2.0, dloss), backward(hn, head, *b, lse, 2.0, dloss)
    for x, y in zip(ga, gb):
        assert bool(((x - y).abs() <= 2.0 ** -20 * x.abs().max()).all())


@pytest.mark.parametrize("t", [20, 150])
def test_bad_rows(t):
    """Tokens out of range or twice and teachers that are not finite: NaN losses without a
    gradient, named by the result; other rows are as without them."""
    hn, head, ids, z, dloss = inputs(t, 64, 500, 10, 11, ragged=False, masked=0.0)
    lse = teacher_lse(ids, z, 1.0)
    want = forward(hn, head, ids, z, lse, 1.0)[0]
    g_want = backward(hn, head, ids, z, lse, 1.0, dloss)[0]
    ids[3, 4], ids[5, 0], ids[7, 9] = 500, -1, ids[7, 2]
    z[9, 1], z[11, 3] = float("nan"), float("inf")
    lse[13] = float("nan")
    ids[15], z[16] = IGN, -math.inf  # without entries
    ids[17, 3], z[17, 3] = 2 ** 40, -math.inf  # not there, whatever its token
    bad = [3, 5, 7, 9, 11, 13]
    loss, res = forward(hn, head, ids, z, lse, 1.0)
    assert int(res[0]) == t - 2 and int(res[1]) == 3
    with pytest.raises(CfattnError, match="row 3 "):
        P.distill_check(res)
    assert bool(torch.isnan(loss[bad]).all()) and loss[15] == 0 and loss[16] == 0
    rest = [i for i in range(t) if i not in (*bad, 15, 16, 17)]
    assert torch.equal(loss[rest], want[rest]) and bool(torch.isfinite(loss[17]))
    dloss[bad] = float("nan")  # (not read)
    keep = kept(hn, head, ids, z, lse, 1.0)
    for k in (None, keep[0]):
        dhn, dhead = backward(hn, head, ids, z, lse, 1.0, dloss, k)
        assert not dhn[bad].any() and not dhn[15:17].any() and bool(torch.isfinite(dhead).all())
        off = (dhn[rest] - g_want[rest]).abs()
        assert bool((off <= 2.0 ** -20 * g_want[rest].abs().amax(1, keepdim=True)).all())


@pytest.mark.parametrize("t", [20, 150])
def test_rows_that_are_not_finite_stay_alone(t):
    hn, head, ids, z, dloss = inputs(t, 64, 500, 10, 11, masked=0.0)
    lse = teacher_lse(ids, z, 1.0)
    want, _ = forward(hn, head, ids, z, lse, 1.0)
    g_want, _ = backward(hn, head, ids, z, lse, 1.0, dloss, want_head=False)
    hn[2, 3], hn[4, 0] = float("nan"), float("inf")
    loss, res = forward(hn, head, ids, z, lse, 1.0)
    P.distill_check(res)
    rest = [i for i in range(t) if i not in (2, 4)]
    assert torch.equal(loss[rest], want[rest]) and bool(torch.isnan(loss[[2, 4]]).all())
    keep = kept(hn, head, ids, z, lse, 1.0)
    for k in (None, keep[0]):
        dhn, _ = backward(hn, head, ids, z, lse, 1.0, dloss, k, want_head=False)
        assert torch.equal(dhn[rest], g_want[rest])


def test_nothing_scored_and_no_rows():
    for t in (10, 100):
        hn, head, ids, z, dloss = inputs(t, 32, 200, 5, 1)
        ids[:] = IGN
        loss, res = forward(hn, head, ids, z, None, 1.0)
        assert not loss.any() and int(res[0]) == 0 and float(P.ce_result_loss(res)) == 0.0
        dhn, dhead = backward(hn, head, ids, z, None, 1.0, dloss)
        assert not dhn.any() and not dhead.any()
        assert bool((backward(hn, head, ids, z, None, 1.0, dloss, acc=True)[1] == 1).all())
    e = torch.empty(0, 32, device=DEV)
    none = torch.empty(0, 5, dtype=torch.int64, device=DEV)
    loss, res = forward(e, head, none, torch.empty(0, 5, device=DEV), None, 1.0)
    assert int(res[0]) == 0 and float(P.ce_result_loss(res)) == 0.0
    assert not backward(e, head, none, torch.empty(0, 5, device=DEV), None, 1.0, loss)[1].any()


def test_chunks_of_rows():
    """Without a keep, logits and exponentials go in chunks that fit the head's limit."""
    hn, head, ids, z, dloss = inputs(700, 48, 1000, 20, 2)
    lse = teacher_lse(ids, z, 1.0)
    want, g = forward(hn, head, ids, z, lse, 1.0)[0], backward(hn, head, ids, z, lse, 1.0, dloss)
    few = [x[:60].contiguous() for x in (hn, ids, z, lse, dloss)]  # (chunks of 33 rows and 27: either product)
    f_want = forward(few[0], head, *few[1:4], 1.0)[0]
    fg = backward(few[0], head, *few[1:4], 1.0, few[4])
    try:
        P.set_head_chunk_limit(128 * 1024 * 4)
        got, h = forward(hn, head, ids, z, lse, 1.0)[0], backward(hn, head, ids, z, lse, 1.0, dloss)
        P.set_head_chunk_limit(33 * 1000 * 4)
        f_got = forward(few[0], head, *few[1:4], 1.0)[0]
        fh = backward(few[0], head, *few[1:4], 1.0, few[4])
    finally:
        P.set_head_chunk_limit(512 << 20)
    assert torch.equal(got, want) and torch.equal(f_got, f_want)
    for x, y in zip((*g, *fg), (*h, *fh)):
        assert bool(((x - y).abs() <= 2.0 ** -20 * x.abs().max()).all())


@pytest.mark.parametrize("t", [30, 200])
def test_another_forwards_keep_gives_nan(t):
    hn, head, ids, z, dloss = inputs(t, 48, 1000, 20, 2)
    n = P.lm_head_distill_keep_bytes(t, 48, 1000, 20)
    keep = torch.zeros(n, dtype=torch.uint8, device=DEV)

    def gives_nan():
        dhn, dhead = backward(hn, head, ids, z, None, 1.0, dloss, keep)
        assert bool(torch.isnan(dhn).all()) and bool(torch.isnan(dhead).all())
    gives_nan()  # (no forward has written it)
    a = inputs(t - 1, 48, 1000, 20, 2)
    forward(*a[:4], None, 1.0, keep)
    gives_nan()
    if t > 64:  # a log-probabilities' keep of the same rows
        logp, lse = torch.empty(t, device=DEV), torch.empty(t, device=DEV)
        P.lm_head_logprobs(hn, head, ids.amax(1).contiguous(), t, 48, 1000, logp, lse, P.ce_result_buffer(DEV), keep)
        gives_nan()


@pytest.mark.parametrize("rows", [(4, 10), (3, 5, 20)])
def test_autograd(rows):
    t, d, vocab, k = torch.Size(rows).numel(), 48, 500, 9
    hn, head, ids, z, dloss = inputs(t, d, vocab, k, 4)
    lse = teacher_lse(ids, z, 1.5)
    w = Exact(hn, head, ids, z, lse, 1.5, dloss)
    h, hd = hn.view(*rows, d).clone().requires_grad_(), head.clone().requires_grad_()
    args = ids.view(*rows, k), z.view(*rows, k).clone().requires_grad_(), lse.view(rows), 1.5
    loss, res = A.lm_head_distill(h, hd, *args)
    assert loss.shape == rows and not res.requires_grad
    both = torch.autograd.grad(loss, (h, hd), dloss.view(rows), retain_graph=True)
    near(both[0].view(t, d), w.dhn, w.tol_dhn, "dhn")
    near(both[1], w.dhead, w.tol_dhead, "dhead")
    again = torch.autograd.grad(loss, (h, hd), dloss.view(rows))
    assert all(torch.equal(a, b) for a, b in zip(both, again))
    (one,) = torch.autograd.grad(A.lm_head_distill(h, head, *args)[0], h, dloss.view(rows))
    (other,) = torch.autograd.grad(A.lm_head_distill(hn.view(*rows, d), hd, *args)[0], hd, dloss.view(rows))
    assert torch.equal(one, both[0]) and torch.equal(other, both[1])
    with torch.no_grad():
        assert torch.equal(A.lm_head_distill(h, hd, *args)[0], loss)


@pytest.mark.parametrize("t", [12, 90])
def test_gradients_against_differences(t):
    """Along a direction that moves no logit by more than 1, (f(+e) - f(-e)) / 2e of the
    forward's losses weighted by dloss: each loss is off by its tolerance, and the third
    derivative of a softmax's logarithm along a change of the logits by v is at most
    (2 |v|_max)^3 a row (twice that with the rest's, of p_rest)."""
    hn, head, ids, z, dloss = inputs(t, 64, 400, 9, 4)
    lse = teacher_lse(ids, z, 1.0, share=0.3)
    w = Exact(hn, head, ids, z, lse, 1.0, dloss)
    grads = backward(hn, head, ids, z, lse, 1.0, dloss)
    g = torch.Generator(device=DEV).manual_seed(1)
    for at, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g, device=DEV)
        v /= float(((v @ head.T) if at == 0 else (hn @ v.T)).abs().max())
        e = 2.0 ** -7

        def f(s):
            a = [hn, head]
            a[at] = a[at] + s * e * v
            return float((forward(*a, ids, z, lse, 1.0)[0].double() * dloss).sum())
        slope = (f(1) - f(-1)) / (2 * e)
        want = float((grad.double() * v).sum())
        room = float(((w.tol_loss * 1.5 / e + 2 * e * e / 6 * 2 ** 3) * dloss.abs()).sum())
        assert abs(slope - want) <= room, (at, slope, want, room)
        assert room < 0.1 * float((grad.double() * v).abs().sum())  # (it tells a gradient from none)


def test_captured_replays_beside_eager_calls():
    """Two captured steps, of few and many rows, replayed in turn with eager calls between."""
    runs = []
    for t, vocab in ((40, 900), (300, 1200)):
        hn, head, ids, z, dloss = inputs(t, 64, vocab, 16, t)
        lse = teacher_lse(ids, z, 2.0)
        n = P.lm_head_distill_keep_bytes(t, 64, vocab, 16)
        keep = torch.empty(n, dtype=torch.uint8, device=DEV)
        out = [torch.empty(t, device=DEV), P.ce_result_buffer(DEV), torch.empty_like(hn), torch.empty_like(head)]

        def step(hn=hn, head=head, ids=ids, z=z, lse=lse, dloss=dloss, out=out, keep=keep, t=t, vocab=vocab):
            P.lm_head_distill(hn, head, ids, z, t, 64, vocab, 16, out[0], out[1], lse, 2.0, keep)
            P.lm_head_distill_backward(hn, head, ids, z, dloss, t, 64, vocab, 16, out[2], out[3], lse, 2.0, keep,
                                       acc=False)
        step()
        torch.cuda.synchronize()
        want = [o.clone() for o in out]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((graph, out, want, step))  # (the graph reads what the step holds)
    for rep in range(3):
        for graph, out, want, _ in runs:
            for o in out:
                o.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o.view(torch.int32), w.view(torch.int32)) for o, w in zip(out, want)), rep
            a = inputs(50 << rep, 80, 2000, 30, rep)
            forward(*a[:4], None, 1.0)
            backward(*a[:4], None, 1.0, a[4])
            torch.cuda.synchronize()


def test_repeatable_and_on_a_side_stream():
    hn, head, ids, z, dloss = inputs(400, 64, 3000, 40, 3)
    lse = teacher_lse(ids, z, 1.0)
    want = forward(hn, head, ids, z, lse, 1.0)[0], *backward(hn, head, ids, z, lse, 1.0, dloss)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = forward(hn, head, ids, z, lse, 1.0)[0], *backward(hn, head, ids, z, lse, 1.0, dloss)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    hn, head, ids, z, dloss = inputs(80, 16, 100, 5, 1)
    loss, res = torch.empty(80, device=DEV), P.ce_result_buffer(DEV)
    ok = dict(hn=hn, head=head, ids=ids, teacher=z, t=80, d=16, vocab=100, k=5, loss=loss, result=res)
    P.lm_head_distill(**ok)
    for change, error in ((dict(hn=hn.half()), TypeError), (dict(ids=ids.int()), TypeError),
                          (dict(ids=ids.cpu()), TypeError),
                          (dict(teacher=z.double()), TypeError), (dict(t=79), ShapeError), (dict(k=4), ShapeError),
                          (dict(teacher_lse=loss[:70]), ShapeError), (dict(temperature=0.0), CfattnError),
                          (dict(temperature=-1.0), CfattnError), (dict(temperature=math.nan), CfattnError),
                          (dict(temperature=math.inf), CfattnError), (dict(temperature=1e-45), CfattnError),
                          (dict(ids=ids.t()), ValueError), (dict(result=loss), TypeError),
                          (dict(keep=torch.empty(64, dtype=torch.uint8, device=DEV)), CfattnError),
                          (dict(keep=loss), TypeError)):
        with pytest.raises(error):
            P.lm_head_distill(**{**ok, **change})
    wide = torch.zeros(80, 1025, dtype=torch.int64, device=DEV)
    with pytest.raises(CfattnError, match="1025"):
        P.lm_head_distill(**{**ok, "ids": wide, "teacher": wide.float(), "k": 1025})
    none = torch.empty(80, 0, dtype=torch.int64, device=DEV)
    with pytest.raises(CfattnError, match="k=0"):
        P.lm_head_distill(**{**ok, "ids": none, "teacher": none.float(), "k": 0})
    assert P.lm_head_distill_keep_bytes(80, 16, 100, 1025) == 0 and P.lm_head_distill_keep_bytes(0, 16, 100, 5) == 0
    args = dict(hn=hn, head=head, ids=ids, teacher=z, dloss=dloss, t=80, d=16, vocab=100, k=5)
    P.lm_head_distill_backward(**args)  # (wants nothing)
    for change, error in ((dict(dhn=hn[:79].clone()), ShapeError), (dict(dhead=head.half()), TypeError),
                          (dict(dloss=dloss[:7]), ShapeError),
                          (dict(dhn=hn.clone(), keep=torch.empty(64, dtype=torch.uint8, device=DEV)), CfattnError)):
        with pytest.raises(error):
            P.lm_head_distill_backward(**{**args, **change})
