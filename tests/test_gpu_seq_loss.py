"""GPU tests of the preference and policy losses (cfops_preference_loss,
cfops_policy_loss) against a plain statement in 64 bits and against differences."""
import numpy as np
import pytest
import torch

from cpuforge_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = -100
EPS = 2.0 ** -24  # half a step of f32


def seqs(lengths, seed, lead=0, tail=3, masked=0.3):
    """Packed sequences with `lead` rows before the first and `tail` behind the
    last: (offsets, targets, logp, ref, old) on the host."""
    r = np.random.RandomState(seed)
    off = lead + np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    rows = int(off[-1]) + tail
    tg = r.randint(0, 1000, rows).astype(np.int64)
    tg[r.rand(rows) < masked] = IGN
    ref = (-5 * r.rand(rows)).astype(np.float32)
    logp = (ref + 0.2 * r.randn(rows)).astype(np.float32)
    old = (logp + 0.2 * r.randn(rows)).astype(np.float32)
    return off, tg, logp, ref, old


def preference(off, tg, logp, ref, beta, form, margin, smooth, mean):
    """(loss, accuracy, margin, rewards, dlogp with NaN in the rows left alone)."""
    n = len(off) - 1
    x = logp.astype(np.float64) - (0 if ref is None else ref.astype(np.float64))
    use = np.ones(len(x), bool) if tg is None else tg != IGN
    rew, share = np.zeros(n), np.zeros(n)
    for i in range(n):
        rows = np.arange(off[i], off[i + 1])
        rows = rows[use[rows]]
        share[i] = beta / max(len(rows), 1) if mean else beta
        rew[i] = share[i] * x[rows].sum()
    diff = rew[::2] - rew[1::2]
    z = diff - margin
    if form == "sigmoid":
        loss = (1 - smooth) * np.logaddexp(0, -z) + smooth * np.logaddexp(0, z)
        dz = 1 / (1 + np.exp(-z)) - (1 - smooth)
    elif form == "hinge":
        loss, dz = np.maximum(0, 1 - z), np.where(z < 1, -1.0, 0.0)
    else:
        loss, dz = (z - 0.5) ** 2, 2 * (z - 0.5)
    d = np.full(len(x), np.nan)
    for i in range(n):
        rows = np.arange(off[i], off[i + 1])
        d[rows] = np.where(use[rows], dz[i // 2] * (-1) ** i * share[i] / (n // 2), 0.0)
    return loss.mean(), (diff > 0).mean(), diff.mean(), rew, d


def run_preference(off, tg, logp, ref, **kw):
    from cpuforge_amd import ops as P
    t = lambda x: None if x is None else torch.from_numpy(x).to(DEV)  # noqa: E731
    d = torch.full((len(logp),), 77.0, device=DEV)
    rew = torch.empty(len(off) - 1, device=DEV)
    res = torch.full((P.PREFERENCE_RESULT_WORDS,), 5, dtype=torch.int32, device=DEV)
    P.preference_loss(t(logp), t(ref), t(tg), t(off), d, rew, res, **kw)
    P.preference_check(res)
    r = P.preference_result(res)
    return float(r.loss), float(r.accuracy), float(r.margin), rew.cpu().numpy(), d.cpu().numpy()


def check_preference(got, want, logp, off, beta):
    loss, acc, margin, rew, d = want
    # 64-bit sums, rounded once; the sums themselves are off by 2^-52 of their terms.
    slack = 2.0 ** -45 * (1 + beta * np.abs(logp.astype(np.float64)).sum())
    assert abs(got[0] - loss) <= EPS * abs(loss) + slack and abs(got[2] - margin) <= EPS * abs(margin) + slack
    assert got[1] == np.float32(acc)
    assert (np.abs(got[3] - rew) <= EPS * np.abs(rew) + slack).all()
    left = np.isnan(d)
    assert (got[4][left] == 77.0).all()
    assert (np.abs(got[4] - d)[~left] <= EPS * np.abs(d[~left]) + slack * np.abs(d[~left]) + 2.0 ** -149).all()


LENGTHS = [[1, 1], [0, 5], [0, 0], [3, 0, 64, 65], [63, 200, 1, 129, 513, 2], [3000, 2500], [17] * 128, [40] * 130,
           [9000, 8000, 1, 700], [70000, 100]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("form,mean", [("sigmoid", False), ("sigmoid", True), ("hinge", False), ("squared", True)])
def test_preference_matches_64_bits(lengths, form, mean):
    print(lengths[:4], form, mean, flush=True)
    off, tg, logp, ref, _ = seqs(lengths, len(lengths) + max(lengths), lead=2)
    for r, g in ((ref, tg), (None, tg), (ref, None)):
        kw = dict(beta=0.3, form=form, margin=0.1, label_smoothing=0.1 if form == "sigmoid" else 0.0)
        got = run_preference(off, g, logp, r, length_mean=mean, **kw)
        check_preference(got, preference(off, g, logp, r, 0.3, form, 0.1, kw["label_smoothing"], mean), logp, off, 0.3)


def test_preference_masked_rows_are_not_read():
    off, tg, logp, ref, _ = seqs([40, 50, 30, 20], 3)
    tg[off[2]:off[3]] = IGN  # one sequence with nothing scored
    want = preference(off, tg, logp, ref, 0.2, "sigmoid", 0.0, 0.0, True)
    logp[tg == IGN], ref[tg == IGN] = np.nan, np.inf
    got = run_preference(off, tg, logp, ref, beta=0.2, length_mean=True)
    check_preference(got, want, np.zeros(1, np.float32), off, 0.2)


def test_preference_of_far_apart_sequences_stays_finite():
    """Rewards thousands apart: the loss is linear, the gradient saturates."""
    off = np.array([0, 100, 200], np.int64)
    logp = np.concatenate([np.full(100, -50.0), np.zeros(100)]).astype(np.float32)
    for sign in (1, -1):
        got = run_preference(off, None, sign * logp, None, beta=1.0)
        want = preference(off, None, sign * logp, None, 1.0, "sigmoid", 0.0, 0.0, False)
        check_preference(got, want, logp, off, 1.0)
        assert np.isfinite(got[0]) and np.isfinite(got[4][:200]).all()


def test_preference_gradient_against_differences():
    off, tg, logp, ref, _ = seqs([20, 30, 7, 12], 4)
    for form, smooth in (("sigmoid", 0.2), ("squared", 0.0)):
        f = lambda lp: preference(off, tg, lp, ref, 0.5, form, 0.1, smooth, False)[0]  # noqa: E731
        d = run_preference(off, tg, logp, ref, beta=0.5, form=form, margin=0.1, label_smoothing=smooth)[4]
        for r in (0, 3, 21, 55, 60):
            h = 1e-5
            up, down = logp.astype(np.float64), logp.astype(np.float64)
            up[r] += h
            down[r] -= h
            # (Differences in 64 bits: h^2 of the third derivative, 2^-52 / h.)
            num = (f(up) - f(down)) / (2 * h)
            assert abs(d[r] - num) <= 1e-8 + EPS * abs(num)


def policy(off, tg, logp, old, ref, adv, per_token, lo, hi, beta, reduction):
    n = len(off) - 1
    use = np.ones(len(logp), bool) if tg is None else tg != IGN
    cnt = np.array([use[off[i]:off[i + 1]].sum() for i in range(n)])
    d, loss, kl, cut = np.full(len(logp), np.nan), 0.0, 0.0, 0
    for i in range(n):
        for r in range(off[i], off[i + 1]):
            d[r] = 0.0
            if not use[r]:
                continue
            w = 1 / cnt.sum() if reduction == "token" else 1 / (cnt[i] * (cnt > 0).sum())
            lp = float(logp[r])
            A = float(adv[r] if per_token else adv[i])
            rt = np.exp(lp - float(old[r])) if old is not None else 1.0
            c = min(max(rt, 1 - lo), 1 + hi)
            past = rt * A > c * A
            loss_r, dr = -min(rt * A, c * A), 0.0 if past else -rt * A
            cut += past
            if ref is not None:
                x = float(ref[r]) - lp
                kl += w * (np.expm1(x) - x)
                loss_r, dr = loss_r + beta * (np.expm1(x) - x), dr - beta * np.expm1(x)
            loss += w * loss_r
            d[r] = w * dr
    return loss, kl, cut / max(cnt.sum(), 1), int(cnt.sum()), d


def run_policy(off, tg, logp, old, ref, adv, **kw):
    from cpuforge_amd import ops as P
    t = lambda x: None if x is None else torch.from_numpy(x).to(DEV)  # noqa: E731
    d = torch.full((len(logp),), 77.0, device=DEV)
    res = torch.full((P.POLICY_RESULT_WORDS,), 5, dtype=torch.int32, device=DEV)
    P.policy_loss(t(logp), t(old), t(ref), t(adv), t(tg), t(off), d, res, **kw)
    P.policy_check(res)
    r = P.policy_result(res)
    return float(r.loss), float(r.kl), float(r.clipped), int(r.n_scored), d.cpu().numpy()


def check_policy(got, want, size):
    """`size` bounds the loss's terms: 64-bit sums in another order, rounded once."""
    slack = 2.0 ** -45 * size
    assert abs(got[0] - want[0]) <= EPS * abs(want[0]) + slack
    assert abs(got[1] - want[1]) <= EPS * abs(want[1]) + slack
    assert abs(got[2] - want[2]) <= EPS * want[2] and got[3] == want[3]
    left = np.isnan(want[4])
    assert (got[4][left] == 77.0).all()
    w = want[4][~left]
    assert (np.abs(got[4][~left] - w) <= (EPS + 2.0 ** -45) * np.abs(w) + 2.0 ** -149).all()


@pytest.mark.parametrize("lengths", [[1], [0], [0, 3, 0], [64, 65, 1], [500, 3, 700], [17] * 65, [9000, 9001],
                                     [30] * 700], ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_matches_64_bits(lengths, reduction):
    print(lengths[:4], reduction, flush=True)
    off, tg, logp, ref, old = seqs(lengths, len(lengths) + max(lengths), lead=1)
    r = np.random.RandomState(7)
    rows, n = len(logp), len(lengths)
    for per_token, use_ref, use_old, g in ((False, True, True, tg), (True, False, True, tg), (True, True, False, None)):
        adv = r.randn(rows if per_token else n).astype(np.float32)
        a = (logp, old if use_old else None, ref if use_ref else None, adv)
        got = run_policy(off, g, *a, clip_low=0.2, clip_high=0.3, kl_coef=0.05, reduction=reduction,
                         per_token=per_token)
        check_policy(got, policy(off, g, *a, per_token, 0.2, 0.3, 0.05, reduction), 20.0)


def test_policy_masked_rows_and_borders():
    """Rows with the ratio just inside, on and just past either border, for
    either sign of the advantage; NaN where nothing is scored."""
    lo, hi = np.log1p(-0.25), np.log1p(0.5)
    old = np.float32(-2.0)
    steps = []
    for b in (lo, hi):
        c = np.float32(old + b)
        steps += [np.nextafter(c, np.float32(-9)), c, np.nextafter(c, np.float32(9))]
    logp = np.array(steps * 2 + [np.nan, np.inf], np.float32)
    adv = np.array([1.0] * 6 + [-1.0] * 6 + [np.nan, 1.0], np.float32)
    tg = np.array([3] * 12 + [IGN, IGN], np.int64)
    olds = np.full(14, old, np.float32)
    off = np.array([0, 14], np.int64)
    want = policy(off, tg, logp, olds, None, adv, True, 0.25, 0.5, 0.0, "token")
    got = run_policy(off, tg, logp, olds, None, adv, clip_low=0.25, clip_high=0.5)
    check_policy(got, want, 20.0)
    assert 0 < want[2] < 1


def test_policy_gradient_against_differences():
    off, tg, logp, ref, old = seqs([20, 30, 7], 4, masked=0.2)
    adv = np.random.RandomState(3).randn(3).astype(np.float32)
    f = lambda lp: policy(off, tg, lp, old, ref, adv, False, 0.2, 0.3, 0.1, "sequence")[0]  # noqa: E731
    d = run_policy(off, tg, logp, old, ref, adv, clip_low=0.2, clip_high=0.3, kl_coef=0.1, reduction="sequence")[4]
    for r in (0, 3, 21, 50, 55):
        h = 1e-5
        up, down = logp.astype(np.float64), logp.astype(np.float64)
        up[r] += h
        down[r] -= h
        num = (f(up) - f(down)) / (2 * h)
        assert abs(d[r] - num) <= 1e-8 + EPS * abs(num)


BAD = [[0, 5, 4, 9, 12], [0, 5, 8, 9, 13], [-1, 5, 8, 9, 12], [0, 5, 8, 2 ** 40, 12], [-2 ** 62, 2 ** 62, 3, 4, 5]]

# Few long sequences, whose rows many workgroups share, beside ones with nothing.
SPLIT = [[40000, 3], [1500, 1700, 0, 1600, 1, 2500, 1200, 900], [8192] * 6, [1023, 1025, 4097, 511, 513, 0, 7000, 2]]


@pytest.mark.parametrize("lengths", SPLIT, ids=lambda x: f"{len(x)}x{max(x)}")
def test_sequences_of_many_workgroups(lengths):
    off, tg, logp, ref, old = seqs(lengths, sum(lengths), lead=5, tail=4)
    tg[off[-2]:off[-1]] = IGN
    for form, mean in (("sigmoid", True), ("squared", False)):
        got = run_preference(off, tg, logp, ref, beta=0.2, form=form, length_mean=mean)
        check_preference(got, preference(off, tg, logp, ref, 0.2, form, 0.0, 0.0, mean), logp, off, 0.2)
    for reduction in ("token", "sequence"):
        for per_token in (True, False):
            adv = np.random.RandomState(5).randn(len(logp) if per_token else len(lengths)).astype(np.float32)
            got = run_policy(off, tg, logp, old, ref, adv, clip_low=0.2, clip_high=0.3, kl_coef=0.05,
                             per_token=per_token, reduction=reduction)
            check_policy(got, policy(off, tg, logp, old, ref, adv, per_token, 0.2, 0.3, 0.05, reduction), 20.0)


def test_bad_offsets_among_many_workgroups():
    off, tg, logp, ref, old = seqs([5000] * 4, 8)
    off[2] = len(logp) + 1  # sequences 1 and 2 do not rise within the rows
    from cpuforge_amd import ops as P
    t = lambda x: torch.from_numpy(x).to(DEV)  # noqa: E731
    d, rew = torch.full((len(logp),), 77.0, device=DEV), torch.empty(4, device=DEV)
    res = torch.empty(P.PREFERENCE_RESULT_WORDS, dtype=torch.int32, device=DEV)
    P.preference_loss(t(logp), t(ref), t(tg), t(off), d, rew, res, beta=0.1)
    with pytest.raises(_lib.CfattnError, match="sequence 1"):
        P.preference_check(res)
    assert P.preference_result(res).loss.isnan() and (d[5000:15000] == 77.0).all()
    pres = torch.empty(P.POLICY_RESULT_WORDS, dtype=torch.int32, device=DEV)
    d.fill_(77.0)
    P.policy_loss(t(logp), t(old), None, torch.ones(4, device=DEV), t(tg), t(off), d, pres, clip_low=0.2, clip_high=0.2)
    with pytest.raises(_lib.CfattnError, match="sequence 1"):
        P.policy_check(pres)
    assert P.policy_result(pres).loss.isnan() and (d[5000:15000] == 77.0).all()


@pytest.mark.parametrize("off", BAD)
def test_offsets_that_do_not_rise_are_not_followed(off):
    from cpuforge_amd import ops as P
    first = next(i for i in range(4) if not 0 <= off[i] <= off[i + 1] <= 12)
    x = torch.zeros(12, device=DEV)
    o = torch.tensor(off, device=DEV)
    res = torch.zeros(8, dtype=torch.int32, device=DEV)
    d = torch.zeros(12, device=DEV)
    P.preference_loss(x, None, None, o, d, torch.empty(4, device=DEV), res, beta=0.1)
    assert bool(torch.isnan(P.preference_result(res).loss))
    with pytest.raises(_lib.CfattnError, match=f"sequence {first} "):
        P.preference_check(res)
    P.policy_loss(x, x, x, torch.ones(4, device=DEV), None, o, d, res, clip_low=0.2, clip_high=0.2)
    assert bool(torch.isnan(P.policy_result(res).loss))
    with pytest.raises(_lib.CfattnError, match=f"sequence {first} "):
        P.policy_check(res)


def test_refusals():
    from cpuforge_amd import ops as P
    x, o = torch.zeros(4, device=DEV), torch.tensor([0, 2, 4], device=DEV)
    res = torch.zeros(8, dtype=torch.int32, device=DEV)
    rew = torch.zeros(2, device=DEV)
    for kw in (dict(label_smoothing=1.0), dict(label_smoothing=-0.1), dict(form="hinge", label_smoothing=0.1)):
        with pytest.raises(_lib.CfattnError, match="label_smoothing"):
            P.preference_loss(x, x, None, o, x, rew, res, beta=0.1, **kw)
    with pytest.raises(_lib.CfattnError, match="pairs"):
        P.preference_loss(x, x, None, o[:1], x, rew[:0], res, beta=0.1)
    with pytest.raises(_lib.ShapeError):
        P.preference_loss(x, x[:3], None, o, x, rew, res, beta=0.1)
    with pytest.raises(TypeError):
        P.preference_loss(x, x, None, o.int(), x, rew, res, beta=0.1)
    for kw in (dict(clip_low=-0.1, clip_high=0.2), dict(clip_low=1.5, clip_high=0.2), dict(clip_low=0.1, clip_high=-1)):
        with pytest.raises(_lib.CfattnError, match="clip"):
            P.policy_loss(x, x, None, rew, None, o, x, res, **kw)
    with pytest.raises(_lib.ShapeError):
        P.policy_loss(x, x, None, torch.zeros(3, device=DEV), None, o, x, res, clip_low=0.1, clip_high=0.1)
    for f in (lambda o: P.policy_loss(x, x, None, x, None, o, x, res, clip_low=0.1, clip_high=0.1),
              lambda o: P.preference_loss(x, x, None, o, x, rew, res, beta=0.1)):
        with pytest.raises(_lib.ShapeError):
            f(o[:0])


def test_captured_losses_replay():
    from cpuforge_amd import ops as P
    off, tg, logp, ref, old = seqs([300, 200, 4000, 100, 9000, 9000], 9)
    t = lambda x: torch.from_numpy(x).to(DEV)  # noqa: E731
    off, tg, lp, ref, old = map(t, (off, tg, logp, ref, old))
    adv = torch.randn(6, device=DEV)

    def step(d, rew, r1, r2):
        P.preference_loss(lp, ref, tg, off, d[0], rew, r1, beta=0.1)
        P.policy_loss(lp, old, ref, adv, tg, off, d[1], r2, clip_low=0.2, clip_high=0.2, kl_coef=0.1)

    def bufs():
        return (torch.zeros(2, lp.numel(), device=DEV), torch.zeros(6, device=DEV),
                torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV))
    a, b = bufs(), bufs()
    step(*b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*a)
    for i in range(4):
        lp.add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        step(*b)
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i


def test_autograd_losses():
    from cpuforge_amd import autograd as A
    off, tg, logp, ref, old = seqs([30, 20, 10, 45], 10, tail=2)
    t = lambda x: torch.from_numpy(x).to(DEV)  # noqa: E731
    lp = t(logp).requires_grad_()
    loss, rewards, _ = A.preference_loss(lp, t(ref), t(tg), t(off), beta=0.1)
    (g,) = torch.autograd.grad(3 * loss, lp)
    want = preference(off, tg, logp, ref, 0.1, "sigmoid", 0.0, 0.0, False)
    w = np.nan_to_num(want[4]) * 3  # rows of no sequence have no gradient
    assert (np.abs(g.cpu().numpy() - w) <= 3 * EPS * np.abs(w) + 1e-12).all()
    assert not rewards.requires_grad
    adv = np.array([1, -1, 0.5, 2], np.float32)
    loss, _ = A.policy_loss(lp, t(old), t(ref), t(adv), t(tg), t(off), clip_low=0.2, clip_high=0.2, kl_coef=0.1)
    (g,) = torch.autograd.grad(loss, lp)
    w = np.nan_to_num(policy(off, tg, logp, old, ref, adv, False, 0.2, 0.2, 0.1, "token")[4])
    assert (np.abs(g.cpu().numpy() - w) <= 2 * EPS * np.abs(w) + 1e-12).all()
