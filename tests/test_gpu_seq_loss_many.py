"""GPU tests of the losses over many thousands of short sequences
(cfops_policy_loss, cfops_preference_loss) against 64 bits."""
import pytest
import torch

from tests.test_gpu_seq_loss import EPS, IGN

pytestmark = pytest.mark.gpu
DEV = "cuda"


def batch(seqs, most, seed):
    """`seqs` sequences of 0 to `most` rows, a third of them not scored."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = torch.randint(0, most + 1, (seqs,), generator=g, device=DEV)
    off = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), n.cumsum(0)])
    rows = int(off[-1])
    tg = torch.randint(0, 1000, (rows,), generator=g, device=DEV)
    tg[torch.rand(rows, generator=g, device=DEV) < 0.33] = IGN
    ref = -5 * torch.rand(rows, generator=g, device=DEV)
    lp = ref + 0.2 * torch.randn(rows, generator=g, device=DEV)
    old = lp + 0.2 * torch.randn(rows, generator=g, device=DEV)
    return off, torch.repeat_interleave(torch.arange(seqs, device=DEV), n), tg, lp, ref, old, g


@pytest.mark.parametrize("seqs,most", [(1024, 3), (1025, 3), (5000, 40), (70000, 5), (300000, 2)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_of_many_sequences_matches_64_bits(seqs, most, reduction):
    from cpuforge_amd import ops as P
    off, seq, tg, lp, ref, old, g = batch(seqs, most, seqs)
    adv = torch.randn(seqs, generator=g, device=DEV)
    d, res = torch.full_like(lp, 77.0), torch.zeros(P.POLICY_RESULT_WORDS, dtype=torch.int32, device=DEV)
    P.policy_loss(lp, old, ref, adv, tg, off, d, res, clip_low=0.2, clip_high=0.3, kl_coef=0.05, reduction=reduction)
    P.policy_check(res)
    use = tg != IGN
    cnt = torch.zeros(seqs, dtype=torch.float64, device=DEV).index_add_(0, seq, use.double())
    w = torch.full_like(cnt, 1 / cnt.sum()) if reduction == "token" else 1 / (cnt.clamp(min=1) * (cnt > 0).sum())
    w = torch.where(use, w[seq], 0.0)
    a, r, x = adv.double()[seq], (lp.double() - old.double()).exp(), ref.double() - lp.double()
    cut = r * a > r.clamp(0.8, 1.3) * a
    loss = -torch.minimum(r * a, r.clamp(0.8, 1.3) * a) + 0.05 * (x.expm1() - x)
    want = w * (torch.where(cut, 0.0, -r * a) - 0.05 * x.expm1())
    got = P.policy_result(res)
    # 64-bit sums of `rows` terms in another order, rounded once.
    slack = 2.0 ** -45 * float((w * loss.abs()).sum() + 1)
    for one, exact in ((got.loss, (w * loss).sum()), (got.kl, (w * (x.expm1() - x)).sum()),
                       (got.clipped, (cut & use).sum() / cnt.sum())):
        assert abs(float(one) - float(exact)) <= EPS * abs(float(exact)) + slack
    assert int(got.n_scored) == int(cnt.sum())
    assert bool(((d.double() - want).abs() <= (EPS + 2.0 ** -45) * want.abs() + 2.0 ** -149).all())


def test_policys_time_grows_no_faster_than_its_sequences():
    """Four times the sequences: four times the work (and a launch's latency, which
    does not grow); the square of it would be sixteen."""
    from cpuforge_amd import ops as P

    def least(seqs):
        off, _, tg, lp, ref, old, g = batch(seqs, 4, 1)
        adv, d = torch.randn(seqs, generator=g, device=DEV), torch.empty_like(lp)
        res, times = torch.zeros(P.POLICY_RESULT_WORDS, dtype=torch.int32, device=DEV), []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            P.policy_loss(lp, old, ref, adv, tg, off, d, res, clip_low=0.2, clip_high=0.3)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    few, many = least(40000), least(160000)
    print(few, many, flush=True)
    assert many < 8 * few


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_captured_policy_of_many_sequences_replays(reduction):
    from cpuforge_amd import ops as P
    off, _, tg, lp, ref, old, g = batch(3000, 20, 2)
    adv = torch.randn(3000, generator=g, device=DEV)

    def step(d, res):
        P.policy_loss(lp, old, ref, adv, tg, off, d, res, clip_low=0.2, clip_high=0.3, kl_coef=0.1, reduction=reduction)

    def bufs():
        return torch.zeros_like(lp), torch.zeros(P.POLICY_RESULT_WORDS, dtype=torch.int32, device=DEV)
    a, b = bufs(), bufs()
    step(*b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*a)
    for i in range(4):
        lp.add_(0.01)
        tg.copy_(tg.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        step(*b)
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i


def test_bad_offsets_among_many_sequences():
    from cpuforge_amd import _lib
    from cpuforge_amd import ops as P
    off, _, tg, lp, ref, old, g = batch(3000, 20, 3)
    off[2001] = lp.numel() + 7  # sequences 2000 and 2001 do not rise within the rows
    d, res = torch.full_like(lp, 77.0), torch.zeros(P.POLICY_RESULT_WORDS, dtype=torch.int32, device=DEV)
    P.policy_loss(lp, old, ref, torch.ones(3000, device=DEV), tg, off, d, res, clip_low=0.2, clip_high=0.3)
    with pytest.raises(_lib.CfattnError, match="sequence 2000 "):
        P.policy_check(res)
    assert P.policy_result(res).loss.isnan() and bool((d[off[2000]:off[2002]] == 77.0).all())
