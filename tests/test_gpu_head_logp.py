"""GPU tests of the targets' log-probabilities through the LM head and their
gradients (cfops_lm_head_logprobs, _backward) against 64 bits."""
import pytest
import torch

from cpuforge_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = -100
U = 2.0 ** -24  # half a step of f32


def inputs(t, d, vocab, seed, masked=0.3, std=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    hn = torch.randn(t, d, generator=g, device=DEV)
    head = torch.randn(vocab, d, generator=g, device=DEV) * (std or 2.0 / d ** 0.5)
    tg = torch.randint(0, vocab, (t,), generator=g, device=DEV)
    tg[torch.rand(t, generator=g, device=DEV) < masked] = IGN
    return hn, head, tg, torch.randn(t, generator=g, device=DEV)


def forward(hn, head, tg, check=True, keep=None):
    from cpuforge_amd import ops as P
    t, d = hn.shape
    logp, lse = (torch.full((t,), 77.0, device=DEV) for _ in range(2))
    res = P.ce_result_buffer(DEV)
    P.lm_head_logprobs(hn, head, tg, t, d, head.shape[0], logp, lse, res, keep)
    if check:
        P.ce_check(res, tg, head.shape[0])
    return logp, lse, res


def backward(hn, head, tg, lse, dlogp, want_head=True, keep=None, acc=True):
    from cpuforge_amd import ops as P
    dhn = torch.full_like(hn, 77.0)
    dhead = torch.ones_like(head) if want_head else None
    P.lm_head_logprobs_backward(hn, head, tg, lse, dlogp, *hn.shape, head.shape[0], dhn, dhead, keep, acc=acc)
    return dhn, dhead


def kept(hn, head, tg):
    """A keep buffer as the forward leaves it, of bytes that are no numbers before."""
    from cpuforge_amd import ops as P
    n = P.lm_head_logprobs_keep_bytes(*hn.shape, head.shape[0])
    if n == 0:
        return None
    keep = torch.full((n + 64,), 255, dtype=torch.uint8, device=DEV)
    forward(hn, head, tg, False, keep[:n])
    assert bool((keep[n:] == 255).all())
    return keep[:n]


def reference(hn, head, tg, dlogp):
    """(logp, lse, dhn, dhead, dlogits) in 64 bits, and a bound on a logit's
    error: the f32 products' (2^-22 of |hn| . |head|; their operands hold 22 bits
    or more, and their sums are f32)."""
    x = hn.double() @ head.double().T
    off = 2.0 ** -22 * (hn.abs().double() @ head.abs().double().T).amax(1)
    use = tg != IGN
    ti = tg.clamp(min=0)
    lse = torch.where(use, torch.logsumexp(x, 1), 0.0)
    logp = torch.where(use, x.gather(1, ti[:, None])[:, 0] - lse, 0.0)
    dx = torch.zeros_like(x).scatter_(1, ti[:, None], 1.0) - torch.softmax(x, 1)
    dx = torch.where(use[:, None], dx * torch.where(use, dlogp.double(), 0.0)[:, None], 0.0)
    return logp, lse, dx @ head.double(), dx.T @ hn.double(), dx, off, x


def check(hn, head, tg, dlogp):
    vocab = head.shape[0]
    logp, lse, res = forward(hn, head, tg)
    w_logp, w_lse, w_dhn, w_dhead, dx, off, x = reference(hn, head, tg, dlogp)
    # A sum of exp over the vocabulary in f32: its longest chain of additions, and
    # each term's rounded argument (up to 2^-24 of the largest difference) and exp.
    chain = vocab / 512 + 24 + 8
    spread = (x.amax(1) - x.amin(1)).clamp(max=104.0)
    tol = off + U * (chain + spread + w_lse.abs() * 2)
    use = tg != IGN
    assert bool(((lse - w_lse).abs() <= torch.where(use, tol, 0.0)).all()), (lse - w_lse).abs().max()
    tol2 = tol + off + U * (w_logp.abs() + 2 * w_lse.abs())
    assert bool(((logp - w_logp).abs() <= torch.where(use, tol2, 0.0)).all()), (logp - w_logp).abs().max()
    n = int(use.sum())
    assert int(res[0]) == n and int(res[1]) == 2 ** 31 - 1
    mean = -float(w_logp.sum()) / max(n, 1)
    assert abs(float(res.view(torch.float32)[2]) - mean) <= float(tol2.max()) + 2.0 ** -23 * abs(mean)
    # exp(x - lse): the errors of both, the difference's rounding and exp's, on
    # every dlogit; then products of 22-bit operands in f32 sums.
    p = dx.abs() + torch.zeros_like(dx).scatter_(1, tg.clamp(min=0)[:, None], 1.0) * (dlogp.abs() * use).double()[:, None]
    rel = (off + tol + U * (spread + 8))[:, None] + 2.0 ** -21 + U * vocab ** 0.5
    floor = 2.0 ** -36 * dlogp.abs().double()[:, None] * use[:, None]  # dlogits below their row's 2^-36
    e = p * rel + floor
    tol_n = e @ head.abs().double() + 1e-37
    tol_h = e.T @ hn.abs().double() + 2.0 ** -24 * (1 + w_dhead.abs()) + U * hn.shape[0] ** 0.5 * (p.T @ hn.abs().double())
    for keep in (None, kept(hn, head, tg)):
        dhn, dhead = backward(hn, head, tg, lse, dlogp, keep=keep)
        assert bool(((dhn - w_dhn).abs() <= tol_n).all()), (dhn - w_dhn).abs().max()
        assert not dhn[~use].any()
        assert bool(((dhead - 1 - w_dhead).abs() <= tol_h + 1e-37).all()), (dhead - 1 - w_dhead).abs().max()
        assert torch.equal(backward(hn, head, tg, lse, dlogp, False, keep)[0], dhn)
        over = backward(hn, head, tg, lse, dlogp, True, keep, acc=False)[1]  # over ones
        assert bool(((over - w_dhead).abs() <= tol_h + 1e-37).all())


SHAPES = [(1, 1, 1), (1, 64, 5), (3, 7, 130), (1, 576, 4097), (5, 576, 2000), (16, 100, 1000), (17, 576, 1000),
          (15, 50, 63), (32, 576, 3000), (33, 40, 128), (64, 33, 4099), (64, 130, 66), (65, 31, 257), (130, 100, 257), (256, 64, 512), (257, 576, 3001), (300, 65, 50),
          (700, 128, 900), (513, 576, 8192), (1000, 16, 20000), (70, 1500, 300), (66, 2100, 300),
          (40, 3, 7)]


@pytest.mark.parametrize("t,d,vocab", SHAPES)
def test_log_probabilities_and_gradients_match_64_bits(t, d, vocab):
    print(t, d, vocab, flush=True)
    check(*inputs(t, d, vocab, t + d + vocab))


def check_forward(hn, head, tg):
    """The forward alone, without and, where there is one, with a keep."""
    from cpuforge_amd import ops as P
    vocab = head.shape[0]
    w_logp, w_lse, _, _, _, off, x = reference(hn, head, tg, torch.zeros(hn.shape[0], device=DEV))
    tol = off + U * (vocab / 512 + 32 + (x.amax(1) - x.amin(1)).clamp(max=104.0) + w_lse.abs() * 2)
    tol = torch.where(tg != IGN, tol, 0.0)
    n = P.lm_head_logprobs_keep_bytes(*hn.shape, vocab)
    for keep in (None, torch.empty(n, dtype=torch.uint8, device=DEV) if n else None):
        logp, lse, _ = forward(hn, head, tg, keep=keep)
        assert bool(((lse - w_lse).abs() <= tol).all()), (lse - w_lse).abs().max()
        assert bool(((logp - w_logp).abs() <= tol + off + U * (w_logp.abs() + 2 * w_lse.abs())).all())


# The forms of the forward by rows (to 16, to 256, 512 or 1024, more), alignment and the
# rounds of workgroups that its tiles of tokens make, at their borders.
FORWARD = [(16, 64, 16385), (17, 64, 16385), (32, 500, 20000), (33, 8, 127), (64, 129, 1000), (65, 577, 3001),
           (128, 129, 129), (129, 129, 257), (384, 576, 4097), (385, 576, 4097), (200, 2050, 1025), (100, 64, 1),
           (97, 1, 300), (383, 68, 20000), (200, 64, 33000), (129, 36, 40000), (257, 40, 66000), (385, 577, 33000),
           (512, 128, 33000), (513, 128, 33000), (1024, 1028, 20000), (1025, 1028, 20000), (256, 257, 33000),
           (257, 257, 33000)]


@pytest.mark.parametrize("t,d,vocab", FORWARD)
@pytest.mark.parametrize("masked", [0.0, 0.9])
def test_forward_of_every_form(t, d, vocab, masked):
    print(t, d, vocab, masked, flush=True)
    check_forward(*inputs(t, d, vocab, t * d + vocab, masked)[:3])


@pytest.mark.parametrize("d", [256, 257])
def test_forward_of_a_head_off_its_alignment(d):
    hn, head, tg, _ = inputs(80, d, 900, 31)
    off = torch.empty(900 * d + 1, device=DEV)[1:].view(900, d)
    check_forward(hn, off.copy_(head), tg)


@pytest.mark.parametrize("t", [40, 200, 500])
def test_forward_where_later_columns_are_larger(t):
    """Weights that grow by 2^10 along a row, whose power of two follows the
    largest value met so far.  (What their pieces lose, 2^-39 of the largest
    |hn| 2^2 times the largest |head| 2^9 in each of 600 products, 2^-19 in all, is
    within the bound of f32 products, 2^-22 of a sum of 20 or more.)"""
    hn, head, tg, _ = inputs(t, 600, 700, 33)
    assert (hn.abs() @ head.abs().T).amin() > 20
    up = torch.exp2(torch.arange(600, device=DEV) / 60)
    check_forward(hn / up, head * up, tg)
    check_forward(hn * up, head / up, tg)
    head[:, 599] *= 3e4
    check_forward(hn, head, tg)
    head[300:310] *= 1e-30
    head[310:320] = 0.0
    check_forward(hn, head, tg)


@pytest.mark.parametrize("t,d", [(30, 96), (90, 96), (700, 96), (700, 1024), (1200, 96)])
def test_what_is_not_scored_or_not_finite_stays_alone_in_every_form(t, d):
    hn, head, tg, _ = inputs(t, d, 20000, 40 + t)
    logp, lse, _ = forward(hn, head, tg)
    off = tg == IGN
    hn2, tg2 = hn.clone(), tg.clone()
    hn2[off] = float("nan")
    first, second, third = (~off).nonzero()[:3, 0].tolist()
    hn2[first, 7], hn2[second, 3], tg2[third] = float("nan"), float("-inf"), 20000
    logp2, lse2, res = forward(hn2, head, tg2, check=False)
    assert int(res[0]) == int((~off).sum()) and int(res[1]) == third
    odd = torch.tensor([first, second, third], device=DEV)
    assert not bool(torch.isfinite(logp2[odd]).any())
    rest = torch.ones(t, dtype=torch.bool, device=DEV)
    rest[odd] = False
    assert torch.equal(logp2[rest], logp[rest]) and torch.equal(lse2[rest], lse[rest])
    # A row of the head that is not finite is in every row's sum.
    head[19990, d - 1] = float("nan")
    assert bool(torch.isnan(forward(hn, head, tg)[1][~off]).all())


@pytest.mark.parametrize("masked", [0.0, 0.97, 1.0])
@pytest.mark.parametrize("t", [9, 400])
def test_masks(t, masked):
    hn, head, tg, g = inputs(t, 96, 777, 5, masked)
    check(hn, head, tg, g)
    logp, lse, _ = forward(hn, head, tg)
    dhn, dhead = backward(hn, head, tg, lse, g)
    # What is not scored is not read.
    off = tg == IGN
    hn2, lse2, g2 = hn.clone(), lse.clone(), g.clone()
    hn2[off], lse2[off], g2[off] = float("nan"), float("inf"), float("nan")
    logp2, lse3, _ = forward(hn2, head, tg)
    dhn2, dhead2 = backward(hn2, head, tg, lse2, g2)
    assert torch.equal(logp, logp2) and torch.equal(lse, lse3)
    assert torch.equal(dhn, dhn2) and torch.equal(dhead, dhead2)


@pytest.mark.parametrize("t", [4, 300])
def test_large_and_small_logits(t):
    """Logits of +-300 (one weight row far above the others), rows of tiny and
    of zero hidden states, weights over a wide range."""
    hn, head, tg, g = inputs(t, 96, 1500, 6)
    head *= torch.logspace(-6, 0, 1500, device=DEV)[:, None]
    head[700] *= 1e3
    hn[0] *= 1e-20
    hn[1] = 0.0
    hn[2] *= 30.0
    tg[:4] = torch.tensor([3, 700, 701, 5], device=DEV)
    check(hn, head, tg, g)


@pytest.mark.parametrize("t", [4, 300])
def test_targets_out_of_range(t):
    from cpuforge_amd import ops as P
    hn, head, tg, g = inputs(t, 64, 900, 7, 0.0)
    want_logp, want_lse, _ = forward(hn, head, tg)
    good_dhn, _ = backward(hn, head, tg, want_lse, g)
    bad = tg.clone()
    bad[1], bad[3] = 900, -1
    logp, lse, res = forward(hn, head, bad, check=False)
    with pytest.raises(_lib.CfattnError, match="target 900 out of range for vocab 900"):
        P.ce_check(res, bad, 900)
    keep = torch.ones(t, dtype=torch.bool, device=DEV)
    keep[1] = keep[3] = False
    assert torch.equal(logp[keep], want_logp[keep]) and bool(torch.isnan(logp[~keep]).all())
    assert torch.equal(lse[keep], want_lse[keep])
    dhn, dhead = backward(hn, head, bad, lse, g)
    assert not dhn[~keep].any() and bool(torch.isfinite(dhead).all())
    # (The rows' order in a product decides no bits of another row.)
    assert torch.equal(dhn[keep], good_dhn[keep])


@pytest.mark.parametrize("t", [4, 300])
def test_a_row_that_is_not_finite_stays_alone(t):
    hn, head, tg, g = inputs(t, 64, 900, 8, 0.0)
    logp, lse, _ = forward(hn, head, tg)
    dhn, _ = backward(hn, head, tg, lse, g, False)
    hn2 = hn.clone()
    hn2[2, 5] = float("nan")
    logp2, lse2, _ = forward(hn2, head, tg)
    dhn2, _ = backward(hn2, head, tg, lse2, g, False)
    keep = torch.arange(t, device=DEV) != 2
    assert bool(torch.isnan(logp2[2])) and bool(torch.isnan(lse2[2])) and bool(torch.isnan(dhn2[2]).any())
    assert torch.equal(logp[keep], logp2[keep]) and torch.equal(dhn[keep], dhn2[keep])


def test_what_another_forward_kept_gives_nan():
    """A keep of another shape is not followed; one whose targets have changed
    since is the forward's."""
    from cpuforge_amd import ops as P
    hn, head, tg, g = inputs(300, 64, 900, 20)
    _, lse, _ = forward(hn, head, tg)
    other = kept(*inputs(700, 64, 1300, 21)[:3])
    assert other.numel() >= P.lm_head_logprobs_keep_bytes(300, 64, 900)
    for acc in (True, False):
        dhn, dhead = backward(hn, head, tg, lse, g, keep=other, acc=acc)
        assert bool(torch.isnan(dhn).all()) and bool(torch.isnan(dhead).all())
    keep = kept(hn, head, tg)
    want = backward(hn, head, tg, lse, g, keep=keep)
    got = backward(hn, head, tg + 10 ** 6, lse, g, keep=keep)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_sizes_past_the_limits_are_refused():
    from cpuforge_amd import ops as P
    from cpuforge_amd.attention import default_context
    ctx, res = default_context(), P.ce_result_buffer(DEV)
    f, b = ctx._lib.cfops_lm_head_logprobs, ctx._lib.cfops_lm_head_logprobs_backward
    for t, d, vocab in ((1 << 24, 8, 8), (8, 1 << 31, 8), (8, 8, 1 << 26)):
        assert f(ctx.handle, None, None, None, t, d, vocab, None, None, res.data_ptr(), None, 0,
                 None) == _lib.ERR_UNSUPPORTED
        assert b(ctx.handle, None, None, None, None, None, t, d, vocab, None, None, 1, None, 0,
                 None) == _lib.ERR_UNSUPPORTED
        assert P.lm_head_logprobs_keep_bytes(t, d, vocab) == 0


def test_no_rows():
    from cpuforge_amd import ops as P
    e = torch.empty(0, device=DEV)
    head = torch.randn(10, 4, device=DEV)
    tg = torch.empty(0, dtype=torch.int64, device=DEV)
    res = P.ce_result_buffer(DEV)
    P.lm_head_logprobs(e, head, tg, 0, 4, 10, e, e, res)
    assert res.tolist() == [0, 2 ** 31 - 1, 0]
    dhead = torch.ones_like(head)
    P.lm_head_logprobs_backward(e, head, tg, e, e, 0, 4, 10, e, dhead)
    assert bool((dhead == 1).all())
    P.lm_head_logprobs_backward(e, head, tg, e, e, 0, 4, 10, e, dhead, acc=False)
    assert not dhead.any()


def test_refusals():
    from cpuforge_amd import ops as P
    hn, head, tg, g = inputs(4, 8, 10, 1)
    res = P.ce_result_buffer(DEV)
    x = torch.zeros(4, device=DEV)
    with pytest.raises(_lib.ShapeError):
        P.lm_head_logprobs(hn, head, tg[:3], 4, 8, 10, x, x, res)
    with pytest.raises(_lib.ShapeError):
        P.lm_head_logprobs(hn, head, tg, 4, 8, 11, x, x, res)
    with pytest.raises(TypeError):
        P.lm_head_logprobs(hn, head, tg.int(), 4, 8, 10, x, x, res)
    with pytest.raises(TypeError):
        P.lm_head_logprobs(hn, head, tg, 4, 8, 10, x, x, res[:2])
    with pytest.raises(TypeError):
        P.lm_head_logprobs(hn.half(), head, tg, 4, 8, 10, x, x, res)
    with pytest.raises(ValueError):
        P.lm_head_logprobs(hn, head.T.contiguous().T, tg, 4, 8, 10, x, x, res)
    n = P.lm_head_logprobs_keep_bytes(300, 8, 10)
    assert P.lm_head_logprobs_keep_bytes(4, 8, 10) == 0 and P.lm_head_logprobs_keep_bytes(300, 0, 10) == 0
    big, tg3 = torch.zeros(300, 8, device=DEV), torch.zeros(300, dtype=torch.int64, device=DEV)
    keep, y = torch.zeros(n + 16, dtype=torch.uint8, device=DEV), torch.zeros(300, device=DEV)
    for bad, what in ((keep[:n - 1], "needed"), (keep[1:], "aligned")):
        with pytest.raises(_lib.CfattnError, match=what):
            P.lm_head_logprobs(big, head, tg3, 300, 8, 10, y, y, res, bad)
        with pytest.raises(_lib.CfattnError, match=what):
            P.lm_head_logprobs_backward(big, head, tg3, y, y, 300, 8, 10, big, None, bad)
    with pytest.raises(TypeError):
        P.lm_head_logprobs(big, head, tg3, 300, 8, 10, y, y, res, keep.float())
    with pytest.raises(_lib.CfattnError, match="positive"):
        P.lm_head_logprobs(hn[:, :0].contiguous(), head[:, :0].contiguous(), tg, 4, 0, 10, x, x, res)


def test_rows_in_chunks_and_repeated_calls_agree():
    """A limit that cuts the backward's rows into chunks changes no bit of the rows'
    gradients, nor does a second run."""
    from cpuforge_amd import ops as P
    hn, head, tg, g = inputs(700, 96, 2000, 12)
    _, lse, _ = forward(hn, head, tg)
    dhn, dhead = backward(hn, head, tg, lse, g)
    again = backward(hn, head, tg, lse, g)
    assert torch.equal(dhn, again[0]) and torch.equal(dhead, again[1])
    P.set_head_chunk_limit(300 * 2000 * 4)
    try:
        logp2, lse2, _ = forward(hn, head, tg)
        dhn2, dhead2 = backward(hn, head, tg, lse2, g)
    finally:
        P.set_head_chunk_limit(512 << 20)
    w = reference(hn, head, tg, g)
    assert bool(((dhn2 - w[2]).abs() <= 2 * (dhn - w[2]).abs().max()).all())
    assert bool(((dhead2 - dhead).abs() <= 2.0 ** -20 * dhead.abs().max()).all())
    # With what the forward keeps, the head's gradient alone goes in passes.
    keep = kept(hn, head, tg)
    one = backward(hn, head, tg, lse, g, keep=keep)
    P.set_head_chunk_limit(0)
    try:
        many = backward(hn, head, tg, lse, g, keep=keep)
        over = backward(hn, head, tg, lse, g, keep=keep, acc=False)[1]
    finally:
        P.set_head_chunk_limit(512 << 20)
    assert torch.equal(one[0], many[0])
    assert bool(((many[1] - dhead).abs() <= 2.0 ** -20 * dhead.abs().max()).all())
    assert bool(((many[1] - 1 - over).abs() <= 2.0 ** -20 * dhead.abs().max()).all())


def test_captured_step_replays():
    from cpuforge_amd import ops as P
    hn, head, tg, g = inputs(300, 96, 3001, 13)
    t, d, vocab = 300, 96, 3001

    def bufs():
        return [torch.zeros(t, device=DEV), torch.zeros(t, device=DEV), P.ce_result_buffer(DEV), torch.zeros_like(hn),
                torch.zeros_like(head)]

    def step(b):
        P.lm_head_logprobs(hn, head, tg, t, d, vocab, b[0], b[1], b[2])
        b[4].zero_()
        P.lm_head_logprobs_backward(hn, head, tg, b[1], g, t, d, vocab, b[3], b[4])
    a, b = bufs(), bufs()
    step(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for i in range(4):
        hn.mul_(1.01)
        tg.copy_(tg.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        step(b)
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i
    # Outgrown scratch of the graph's stays: a larger eager call, then a replay.
    forward(*inputs(900, 128, 5000, 14)[:3])
    graph.replay()
    step(b)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_autograd():
    from cpuforge_amd import autograd as A
    hn, head, tg, g = inputs(60, 48, 500, 15)
    h3 = hn.view(4, 15, 48).requires_grad_()
    w = head.clone().requires_grad_()
    logp, res = A.lm_head_logprobs(h3, w, tg.view(4, 15))
    assert logp.shape == (4, 15) and not res.requires_grad
    dh, dw = torch.autograd.grad(logp, (h3, w), g.view(4, 15))
    _, lse, _ = forward(hn, head, tg)
    want = backward(hn, head, tg, lse, g, keep=kept(hn, head, tg))
    assert torch.equal(dh.view(60, 48), want[0])
    assert torch.equal(dw, backward(hn, head, tg, lse, g, keep=kept(hn, head, tg), acc=False)[1])
    (only,) = torch.autograd.grad(A.lm_head_logprobs(h3.detach(), w, tg.view(4, 15))[0], w, g.view(4, 15))
    assert torch.equal(only, dw)


def test_autograd_keeps_up_to_its_limit(monkeypatch):
    """With and without what the forward keeps: the same gradients to f32 sums in
    another order; a second backward of one graph gives the first one's."""
    from cpuforge_amd import autograd as A
    hn, head, tg, g = inputs(700, 96, 2000, 17)
    hn.requires_grad_()
    logp, _ = A.lm_head_logprobs(hn, head, tg)
    (a,) = torch.autograd.grad(logp, hn, g, retain_graph=True)
    (b,) = torch.autograd.grad(logp, hn, g)
    assert torch.equal(a, b)
    monkeypatch.setattr(A, "LOGPROBS_KEEP_LIMIT", 1000)
    (c,) = torch.autograd.grad(A.lm_head_logprobs(hn, head, tg)[0], hn, g)
    assert bool(((a - c).abs() <= 2.0 ** -20 * a.abs().max()).all())


def test_against_differences():
    """The gradient against central differences of the 64-bit formula."""
    hn, head, tg, g = inputs(6, 10, 40, 16, 0.2)
    _, lse, _ = forward(hn, head, tg)
    dhn, dhead = backward(hn, head, tg, lse, g)

    def f(h, w):
        return float((reference(h, w, tg, g)[0] * g.double()).sum())
    h64, w64 = hn.double(), head.double()
    for arr, got, at in ((h64, dhn, (0, 3)), (h64, dhn, (4, 9)), (w64, dhead - 1, (3, 2)), (w64, dhead - 1, (39, 0))):
        eps = 1e-6
        keep = float(arr[at])
        arr[at] = keep + eps
        up = f(h64, w64)
        arr[at] = keep - eps
        down = f(h64, w64)
        arr[at] = keep
        num = (up - down) / (2 * eps)
        assert abs(float(got[at]) - num) <= 1e-5 * (1 + abs(num))
