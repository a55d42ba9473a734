"""GPU tests of the gradients of cfops_lm_head_logprobs where a head is uneven:
rows of rare tokens, rows of zeros, tiny rows, one row far above the others.  Each
value is held to the errors of its own terms in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = -100
U = 2.0 ** -24  # half a step of f32


def forward(hn, head, tg, keeps):
    from cpuforge_amd import ops as P
    t, d, vocab = *hn.shape, head.shape[0]
    logp, lse = torch.empty(t, device=DEV), torch.empty(t, device=DEV)
    n = P.lm_head_logprobs_keep_bytes(t, d, vocab) if keeps else 0
    keep = torch.full((n,), 255, dtype=torch.uint8, device=DEV) if n else None
    P.lm_head_logprobs(hn, head, tg, t, d, vocab, logp, lse, P.ce_result_buffer(DEV), keep)
    return logp, lse, keep


def gradients(hn, head, tg, dlogp, keeps):
    from cpuforge_amd import ops as P
    _, lse, keep = forward(hn, head, tg, keeps)
    dhn, dhead = torch.empty_like(hn), torch.empty_like(head)
    P.lm_head_logprobs_backward(hn, head, tg, lse, dlogp, *hn.shape, head.shape[0], dhn, dhead, keep, acc=False)
    return dhn.double(), dhead.double()


def group_top(w, n=32):
    """Each row's largest magnitude of its group of n rows."""
    pad = torch.nn.functional.pad(w.abs(), (0, 0, 0, -len(w) % n))
    return pad.view(-1, n, w.shape[1]).amax((1, 2)).repeat_interleave(n)[:len(w), None]


class Exact:
    """The formulas in 64 bits, and bounds from the products' own: operands of 22
    bits whose last ones lie 2^-39 below the largest value of a row of hn or of 32 rows
    of the head, and f32 sums."""

    def __init__(self, hn, head, tg, dlogp):
        h, w, g = hn.double(), head.double(), dlogp.double()
        use = tg != IGN
        ti = tg.clamp(min=0)
        hot = torch.zeros(len(h), len(w), dtype=torch.float64, device=DEV).scatter_(1, ti[:, None], 1.0)
        x = h @ w.T
        self.P = torch.softmax(x, 1) * use[:, None]
        lse = torch.logsumexp(x, 1)
        dx = (hot * use[:, None] - self.P) * torch.where(use, g, 0.0)[:, None]
        self.dhn, self.dhead = dx @ w, dx.T @ h
        top_h, top_w = h.abs().amax(1, keepdim=True), group_top(w)
        off = 2.0 ** -22 * (h.abs() @ w.abs().T) \
            + h.abs() @ torch.minimum(w.abs(), 2.0 ** -39 * top_w).T \
            + torch.minimum(h.abs(), 2.0 ** -39 * top_h) @ w.abs().T
        # lse: its logits, each weighted by its share; the sum of exp in f32; its own
        # rounding, and that of the exponentials' arguments.
        spread = (x.amax(1) - x.amin(1)).clamp(max=104.0)
        e_lse = (self.P * off).sum(1) + U * (len(w) / 512 + 32 + spread + 2 * lse.abs())
        self.rel = off + (e_lse + U * (spread + 8))[:, None] + 2.0 ** -21
        self.p = (self.P + hot * use[:, None]) * torch.where(use, g, 0.0).abs()[:, None]
        self.h, self.w = h.abs(), w.abs()

    def dhead_bound(self):
        """Sums over tokens, one addition to 16 of them; dlogits as two f16 pieces of
        their column's largest term."""
        n = len(self.h)
        terms = self.p * self.h.amax(1, keepdim=True)
        return (self.p * self.rel).T @ self.h + U * (n / 16 + 16) * (self.p.T @ self.h) \
            + 2.0 ** -38 * n * terms.amax(0)[:, None] + U * self.dhead.abs() + 2.0 ** -126

    def dhn_bound(self):
        """Sums over the vocabulary; probabilities as two f16 pieces that lose 2^-33 of
        the largest of 128 rows of the head, in products with rows of 32."""
        v = len(self.w)
        group = torch.nn.functional.pad(self.P, (0, -v % 128)).view(len(self.h), -1, 128).amax(2)
        group = group.repeat_interleave(128, 1)[:, :v] * self.p.amax(1, keepdim=True).clamp(max=1e30)
        return (self.p * self.rel) @ self.w + U * (v / 64 + 32) * (self.p @ self.w) \
            + 2.0 ** -33 * (group @ self.w) + self.p @ torch.minimum(self.w, 2.0 ** -39 * group_top(self.w)) \
            + U * self.dhn.abs() + 2.0 ** -126


def report(name, err, bound, want):
    rows = (err.norm(dim=1) / want.norm(dim=1).clamp(min=1e-300)).sort().values
    print(f"{name}: of its bound {float((err / bound).max()):.3f}; rows' relative error, median "
          f"{float(rows[len(rows) // 2]):.1e}, worst {float(rows[-1]):.1e}", flush=True)


def check(hn, head, tg, dlogp, keeps, dhn_too=True):
    want = Exact(hn, head, tg, dlogp)
    dhn, dhead = gradients(hn, head, tg, dlogp, keeps)
    err, bound = (dhead - want.dhead).abs(), want.dhead_bound()
    report("dhead", err, bound, want.dhead)
    assert bool((err <= bound).all())
    if dhn_too:
        err, bound = (dhn - want.dhn).abs(), want.dhn_bound()
        report("dhn", err, bound, want.dhn)
        assert bool((err <= bound).all())
    return want, dhn, dhead


def inputs(t, d, vocab, seed, masked=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    hn = torch.randn(t, d, generator=g, device=DEV)
    head = torch.randn(vocab, d, generator=g, device=DEV) * (1.0 / d ** 0.5)
    tg = torch.randint(0, vocab, (t,), generator=g, device=DEV)
    tg[torch.rand(t, generator=g, device=DEV) < masked] = IGN
    return hn, head, tg, torch.randn(t, generator=g, device=DEV)


FORMS = [(60, False), (300, False), (300, True), (700, True)]  # rows, and whether the forward keeps


@pytest.mark.parametrize("t,keeps", FORMS)
@pytest.mark.parametrize("gap", [0, 10, 15, 20, 30, 55])
def test_rare_tokens_rows_of_the_heads_gradient(t, keeps, gap):
    """Half of the head's rows, in among the others, have logits that lie `gap` below
    theirs: their gradients are as exact, of their own size, as the others'."""
    print(t, keeps, gap, flush=True)
    hn, head, tg, g = inputs(t, 64, 2000, 100 + gap)
    hn[:, 0] = 4.0
    rare = torch.rand(2000, generator=torch.Generator().manual_seed(gap)).to(DEV) < 0.5
    head[:, 0] = torch.where(rare, -gap / 4, 0.0)
    tg[tg != IGN] = (~rare).nonzero()[:, 0][tg[tg != IGN] % int((~rare).sum())]
    tg[7] = int(rare.nonzero()[3, 0])
    want, _, dhead = check(hn, head, tg, g, keeps)
    rows = rare & (want.P.sum(0) > 0)
    off = (dhead - want.dhead)[rows].norm(dim=1) / want.dhead[rows].norm(dim=1)
    assert float(off.max()) <= 1e-4 and float(off.median()) <= 1e-5


@pytest.mark.parametrize("t,keeps", FORMS)
def test_heads_gradient_of_zero_and_of_tiny_rows(t, keeps):
    """Rows of the head that are zeros (new or padded entries of a vocabulary) or
    tiny, whole groups of them and single ones: their probabilities are like any
    other's, and so are their gradients."""
    hn, head, tg, g = inputs(t, 64, 1500, 7)
    head[320:384] = 0.0
    head[400:403] = 0.0
    head[416:448] *= 1e-12
    head[448:480] *= 1e-35
    head[640:768] = 0.0
    head[1472:] = 0.0
    want, _, dhead = check(hn, head, tg, g, keeps)
    assert float(want.dhead[320:384].abs().amin(1).min()) > 0
    assert bool((dhead[1472:].abs().amax(1) > 0).all())


@pytest.mark.parametrize("t,keeps", FORMS)
def test_heads_gradient_beside_one_large_row(t, keeps):
    """One row of the head 2^25 times the others (with hidden states that meet it in
    a small component, a logit of -32; its group of 32 rows holds nothing else)."""
    hn, head, tg, g = inputs(t, 64, 1500, 8)
    hn[:, 0] = -2.0 ** -20
    head[:, 0] = 0.0
    head[480:512] = 0.0
    head[500, 0] = 2.0 ** 25
    tg[(tg >= 480) & (tg < 512)] = 3
    check(hn, head, tg, g, keeps, dhn_too=False)


@pytest.mark.parametrize("scale", [1e-6, 1e-20, 1e20])
@pytest.mark.parametrize("t,keeps", FORMS)
def test_heads_gradient_of_small_and_large_hidden_states(t, keeps, scale):
    """Hidden states of any size, the head's gradient of theirs; one row of them
    below all others."""
    hn, head, tg, g = inputs(t, 64, 1500, 9)
    hn[5] *= 1e-8
    check(hn * scale, head / scale, tg, g, keeps)


@pytest.mark.parametrize("t,keeps", FORMS)
@pytest.mark.parametrize("row", [0, 500, 1499])
def test_hidden_states_gradient_beside_one_large_row(t, keeps, row):
    """One row of the head 2^25 times the others, alone in its group of 32, with a
    logit of -32: it moves its own column alone."""
    hn, head, tg, g = inputs(t, 64, 1500, 8)
    hn[:, 0] = -2.0 ** -20
    head[:, 0] = 0.0
    head[row // 32 * 32:row // 32 * 32 + 32] = 0.0
    head[row, 0] = 2.0 ** 25
    tg[tg == row] = 700
    check(hn, head, tg, g, keeps)


@pytest.mark.parametrize("t,keeps", FORMS)
def test_gradients_where_the_heads_size_changes_from_row_to_row(t, keeps):
    """Groups of 32 rows of the head 2^-60 to 1 times the others, in any order, so
    that sums over the vocabulary end and begin in among 128 rows."""
    hn, head, tg, g = inputs(t, 64, 1500, 10)
    size = torch.randint(-60, 1, (47,), generator=torch.Generator().manual_seed(3)).to(DEV)
    head *= torch.exp2(size.float()).repeat_interleave(32)[:1500, None]
    check(hn, head, tg, g, keeps)
    head *= 2.0 ** -90
    check(hn * 2.0 ** 45, head * 2.0 ** 45, tg, g, keeps)


@pytest.mark.parametrize("keeps", [True, False])
def test_scratch_of_the_hidden_states_gradient_is_bounded(keeps):
    """Many rows of a small vocabulary: 512 MiB for the product's partial sums (and,
    with nothing kept, 4 bytes a value of the hidden states and a chunk of the logits),
    their gradient right in every pass."""
    from cpuforge_amd import ops as P
    from cpuforge_amd.attention import Context
    t, d, vocab = 20000, 2048, 300
    hn, head, tg, g = inputs(t, d, vocab, 11)
    want = Exact(hn, head, tg, g)
    bound, exact = want.dhn_bound(), want.dhn
    del want
    _, lse, keep = forward(hn, head, tg, keeps)
    dhn = torch.empty_like(hn)
    ctx = Context(0)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    P.lm_head_logprobs_backward(hn, head, tg, lse, g, t, d, vocab, dhn, None, keep, ctx=ctx)
    torch.cuda.synchronize()
    took = free - torch.cuda.mem_get_info()[0]
    print(took >> 20, "MiB", flush=True)
    assert took <= (560 << 20) + (0 if keeps else 4 * t * (d + 512))
    assert bool(((dhn.double() - exact).abs() <= bound).all())


@pytest.mark.parametrize("keeps", [True, False])
@pytest.mark.parametrize("masked", [0.0, 0.7, 1.0])
def test_passes_with_few_or_no_scored_rows(keeps, masked):
    """Three passes of rows, of which the scored ones fill three, one or none."""
    hn, head, tg, g = inputs(5000, 8192, 300, 12, masked)
    want = Exact(hn, head, tg, g)
    dhn, dhead = gradients(hn, head, tg, g, keeps)
    assert bool(((dhn - want.dhn).abs() <= want.dhn_bound()).all()) and not dhn[tg == IGN].any()
    assert bool(((dhead - want.dhead).abs() <= want.dhead_bound()).all())


@pytest.mark.parametrize("t,d", [(60, 96), (700, 96), (5000, 8192)])
def test_captured_gradients_replay_with_what_the_forward_keeps(t, d):
    """Forward and both gradients in one graph, whose keep is written anew by every
    replay, with eager calls of the same context between the replays."""
    from cpuforge_amd import ops as P
    hn, head, tg, g = inputs(t, d, 300, 13)
    n = P.lm_head_logprobs_keep_bytes(t, d, 300)

    def bufs():
        keep = torch.zeros(n, dtype=torch.uint8, device=DEV) if n else None
        return torch.zeros(t, device=DEV), torch.zeros(t, device=DEV), torch.zeros_like(hn), torch.zeros_like(head), keep

    def step(b):
        logp, lse, dhn, dhead, keep = b
        P.lm_head_logprobs(hn, head, tg, t, d, 300, logp, lse, res, keep)
        P.lm_head_logprobs_backward(hn, head, tg, lse, g, t, d, 300, dhn, dhead, keep, acc=False)
    res = P.ce_result_buffer(DEV)
    a, b = bufs(), bufs()
    step(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for i in range(4):
        hn.mul_(0.99)
        tg.copy_(tg.roll(7))
        graph.replay()
        torch.cuda.synchronize()
        step(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4])), i
