"""GPU tests of preference and policy training steps as a whole: a small
SmolLM-shaped model's log-probabilities, a loss over packed sequences, the
backward into every adapter and an AdamW step with 8-bit moments, against the
same step of the torch backend; and such a step captured in a HIP graph."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from cpuforge_amd import autograd as A
from cpuforge_amd import ops as P
from cpuforge_amd.optim import AdamW, State8
from cpuforge_amd.train_bench import SmolLM
from tests import adamw8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB, SEQ, BATCH = 1000, 64, 6


def models(train="lora"):
    kw = dict(layers=2, seq=SEQ, rank=16 if train == "lora" else 0, config={"vocab": VOCAB}, train=train)
    a, b = SmolLM(backend="cfops", **kw), SmolLM(backend="torch", **kw)
    gen = torch.Generator(device=DEV).manual_seed(4)
    with torch.no_grad():  # adapters some steps into training
        for (_, p), (_, q) in zip(a.named_params(), b.named_params()):
            if p.requires_grad:
                p.add_(torch.randn(p.shape, generator=gen, device=DEV) * 0.02)
            q.copy_(p)
    return a, b


def batch():
    gen = torch.Generator(device=DEV).manual_seed(5)
    tokens = torch.randint(0, VOCAB, (BATCH, SEQ), generator=gen, device=DEV)
    targets = torch.roll(tokens, -1, 1)
    targets[:, -1] = P.IGNORE_INDEX
    for i in range(BATCH):
        targets[i, :3 * i] = P.IGNORE_INDEX  # prompts
        targets[i, SEQ - i:] = P.IGNORE_INDEX  # padding
    offsets = torch.arange(0, BATCH * SEQ + 1, SEQ, device=DEV)
    ref = -7.0 + torch.randn(BATCH * SEQ, generator=gen, device=DEV)
    return tokens, targets, offsets, ref


def torch_logprobs(model, tokens, targets):
    logits = model.hidden(tokens) @ model.embed.t()
    lp = -F.cross_entropy(logits.view(-1, VOCAB), targets.view(-1), ignore_index=P.IGNORE_INDEX, reduction="none")
    return lp  # 0 where ignored


def losses(kind, logp, ref, targets, offsets, lib):
    lp = logp.reshape(-1)
    if kind == "preference":
        if lib:
            return A.preference_loss(lp, ref, targets.view(-1), offsets, beta=0.3, label_smoothing=0.1)[0]
        use = (targets.view(-1) != P.IGNORE_INDEX).float()
        s = 0.3 * ((lp - ref) * use).view(BATCH // 2, 2, SEQ).sum(-1)
        z = s[:, 0] - s[:, 1]
        return -(0.9 * F.logsigmoid(z) + 0.1 * F.logsigmoid(-z)).mean()
    old = lp.detach() + 0.1 * torch.sin(torch.arange(lp.numel(), device=DEV))
    adv = torch.linspace(-1, 1.5, BATCH, device=DEV)
    if lib:
        return A.policy_loss(lp, old, ref, adv, targets.view(-1), offsets, clip_low=0.05, clip_high=0.07, kl_coef=0.1,
                             reduction="sequence")[0]
    use = (targets.view(-1) != P.IGNORE_INDEX).float()
    r = (lp - old).exp()
    a = adv.repeat_interleave(SEQ)
    x = ref - lp
    row = -torch.minimum(r * a, r.clamp(0.95, 1.07) * a) + 0.1 * (x.exp() - x - 1)
    n = use.view(BATCH, SEQ).sum(1)
    return ((row * use).view(BATCH, SEQ).sum(1) / n).mean()


@pytest.mark.parametrize("train", ["lora", "full"])
@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_step_matches_the_torch_backend(kind, train):
    a, b = models(train)
    tokens, targets, offsets, ref = batch()
    logp = a.logprobs(tokens, targets)
    a.check_targets()
    want_logp = torch_logprobs(b, tokens, targets)
    # (Both are f32 models: as the loss of the two backends elsewhere, to 1e-5 of its size.)
    assert bool(((logp.view(-1) - want_logp).abs() <= 1e-5 * (1 + want_logp.abs())).all())
    loss = losses(kind, logp, ref, targets, offsets, True)
    want = losses(kind, want_logp, ref, targets, offsets, False)
    assert abs(float(loss) - float(want)) <= 1e-4 * (1 + abs(float(want)))
    loss.backward()
    want.backward()
    for (name, p), (_, q) in zip(a.named_params(), b.named_params()):
        if p.requires_grad:  # the gradcheck metric of the reference's tests
            worst = ((p.grad - q.grad).abs() / (1 + q.grad.abs())).max()
            assert worst <= 1e-4, (name, float(worst))
    # The optimizer's step from these gradients, its moments in 8 bits.
    opt = AdamW(0.9, 0.99, 1e-8, 0.1, state_bits=8)
    before = {n: p.detach().cpu().numpy().astype(np.float64).reshape(-1) for n, p in a.named_params() if p.requires_grad}
    opt.update(a, 1e-3)
    for name, p in a.named_params():
        if not p.requires_grad:
            continue
        g = p.grad.cpu().numpy().astype(np.float64).reshape(-1)
        z = np.zeros_like(g)
        wd = 0.0 if "norm" in name else 0.1
        p1, m1, v1 = R.step(before[name], g, z, z, 1, 1e-3, 0.9, 0.99, 1e-8, wd)
        got = p.detach().cpu().numpy().astype(np.float64).reshape(-1)
        # p's rounding, and some ten f32 roundings of an update of at most lr (1 + wd |p|).
        assert np.abs(got - p1).max() <= 2.0 ** -24 * np.abs(p1).max() + 10 * 2.0 ** -24 * 1e-3 * (1 + np.abs(p1).max())
        s = opt.state[name]
        assert isinstance(s, State8) == (p.numel() >= 4096)
        if isinstance(s, State8):
            m, v = s.moments()
            assert np.array_equal(m.cpu().numpy().reshape(-1).astype(np.float64), np.float32(m1).astype(np.float64))
            assert np.array_equal(v.cpu().numpy().reshape(-1).astype(np.float64), np.float32(v1).astype(np.float64))


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_captured_step_replays(kind):
    """The step's gradients of every replay are the eager step's, bit for bit,
    with eager work between the replays."""
    a, _ = models()
    tokens, targets, offsets, ref = batch()
    params = a.params()

    def step():
        for p in params:
            p.grad = None
        loss = losses(kind, a.logprobs(tokens, targets), ref, targets, offsets, True)
        loss.backward()
        return loss
    loss = step()
    want_loss, want = loss.detach().clone(), [p.grad.clone() for p in params]
    del loss  # (no eager graph of these leaves lives while the step is captured)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = step()
        del loss
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p in params:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(3):
        graph.replay()
        torch.cuda.synchronize()
        a.check_targets()
        assert torch.equal(got.detach(), want_loss), rep
        assert all(torch.equal(p.grad, w) for p, w in zip(params, want)), rep
        # Eager work of the same operators on the same context, larger and smaller.
        for t in (20, 900 << rep):
            hn, head = torch.randn(t, 64, device=DEV, requires_grad=True), torch.randn(3000, 64, device=DEV, requires_grad=True)
            lp, _ = A.lm_head_logprobs(hn, head, torch.zeros(t, dtype=torch.int64, device=DEV))
            lp.sum().backward()
        torch.cuda.synchronize()


def test_two_streams_one_after_the_other():
    """A call on a side stream, ordered by events, sees the tensors of another."""
    a, _ = models()
    tokens, targets, offsets, ref = batch()
    with torch.no_grad():
        want = a.logprobs(tokens, targets).clone()
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = a.logprobs(tokens, targets)
            d, res = torch.zeros(BATCH * SEQ, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
            P.preference_loss(got.view(-1), ref, targets.view(-1), offsets, d, torch.empty(BATCH, device=DEV), res,
                              beta=0.1)
        side.synchronize()
    assert torch.equal(got, want) and bool(torch.isfinite(P.preference_result(res).loss)) and bool(d.any())


def test_logprobs_of_the_torch_backend_are_refused():
    _, b = models()
    tokens, targets, _, _ = batch()
    with pytest.raises(ValueError, match="cfops"):
        b.logprobs(tokens, targets)
