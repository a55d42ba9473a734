"""GPU tests of a distillation step as a whole: a small model with layer norms,
pairs side by side in half of each head, a scaled RoPE table and several documents
to a row, trained on a teacher's top logits with an AdamW of 8-bit moments, against
the same step in torch operations; and such a step captured in a HIP graph."""
import pytest
import torch

from cpuforge_amd import YarnScaling
from cpuforge_amd import ops as P
from cpuforge_amd.optim import AdamW
from cpuforge_amd.train_bench import SmolLM

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB, SEQ, BATCH, K = 900, 48, 5, 12
CONFIG = dict(vocab=VOCAB, norm="layer", rotary=dict(dim=32, interleaved=True), rope_scaling=YarnScaling(4.0, 24))


def models(train="lora", **config):
    kw = dict(layers=2, seq=SEQ, rank=8 if train == "lora" else 0, config=dict(CONFIG, **config), train=train)
    a, b = SmolLM(backend="cfops", **kw), SmolLM(backend="torch", **kw)
    gen = torch.Generator(device=DEV).manual_seed(4)
    with torch.no_grad():  # some steps into training
        for (_, p), (_, q) in zip(a.named_params(), b.named_params()):
            if p.requires_grad or "norm" in _:
                p.add_(torch.randn(p.shape, generator=gen, device=DEV) * 0.02)
            q.copy_(p)
    return a, b


def batch():
    gen = torch.Generator(device=DEV).manual_seed(5)
    tokens = torch.randint(0, VOCAB, (BATCH, SEQ), generator=gen, device=DEV)
    positions = torch.arange(SEQ, device=DEV).expand(BATCH, SEQ) % 20
    ids = torch.rand(BATCH, SEQ, VOCAB, generator=gen, device=DEV).topk(K).indices
    z = 4 - torch.arange(K, device=DEV) * 0.4 + 0.3 * torch.randn(BATCH, SEQ, K, generator=gen, device=DEV)
    ids[:, ::7] = P.IGNORE_INDEX  # rows without entries
    ids[:, 1::5, 6:] = P.IGNORE_INDEX  # shorter lists
    lse = torch.where(ids == P.IGNORE_INDEX, -torch.inf, z / 2.0).logsumexp(-1).nan_to_num(neginf=0.0) + 0.2
    return tokens, positions.contiguous(), ids, z, lse


def torch_losses(model, tokens, positions, ids, z, lse, temp):
    x = model.hidden(tokens, positions) @ model.embed.t() / temp
    log_q = x.log_softmax(-1)
    there = ids != P.IGNORE_INDEX
    at = ids.clamp(min=0)
    log_p = z / temp - lse[..., None]
    p = torch.where(there, log_p.exp(), 0.0)
    loss = torch.where(there, p * (log_p - log_q.gather(-1, at)), 0.0).sum(-1)
    named = torch.zeros_like(x).scatter_add_(-1, at, there.float()) > 0
    rest = log_q.masked_fill(named, -torch.inf).logsumexp(-1)
    left = 1 - p.sum(-1)
    return torch.where(there.any(-1), loss + left * (left.log() - rest), 0.0)


@pytest.mark.parametrize("train", ["lora", "full"])
def test_step_matches_torch_operations(train):
    a, b = models(train)
    args = batch()
    got = a.distill(args[0], *args[2:], 2.0, positions=args[1])
    a.check_targets()
    want = torch_losses(b, *args, 2.0)
    # (Both are f32 models: as the other steps' tests, to 1e-5 of a logarithm's size and the
    # rest's share, 1 - sum p in f32, by some 2^-22 of 1 over its 0.18.)
    assert bool(((got - want).abs() <= 1e-5 * (1 + want.abs())).all()), float((got - want).abs().max())
    assert not got[:, ::7].any()
    got.sum().backward()
    want.sum().backward()
    for (name, p), (_, q) in zip(a.named_params(), b.named_params()):
        if p.requires_grad:  # the gradcheck metric of the reference's tests
            worst = ((p.grad - q.grad).abs() / (1 + q.grad.abs())).max()
            assert worst <= 1e-4, (name, float(worst))
    if train == "full":
        assert a.final_norm_b.grad.any() and a.layers[0]["attn_norm_b"].grad.any()
    before = [p.detach().clone() for p in a.params()]
    AdamW(0.9, 0.99, 1e-8, 0.1, state_bits=8).update(a, 1e-3)
    for p, was in zip(a.params(), before):
        assert bool(torch.isfinite(p).all()) and not torch.equal(p, was)


def test_captured_step_replays():
    """The step's losses and gradients of every replay are the eager step's, bit for
    bit, with eager work between the replays."""
    a, _ = models()
    tokens, positions, ids, z, lse = batch()
    params = a.params()

    def step():
        for p in params:
            p.grad = None
        loss = a.distill(tokens, ids, z, lse, 2.0, positions=positions)
        loss.sum().backward()
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
        # Eager work of the same operators on the same context.
        x = torch.randn(300 << rep, 576, device=DEV)
        y, s = torch.empty_like(x), torch.empty(2, len(x), device=DEV)
        w = torch.ones(576, device=DEV)
        P.layernorm_forward(x, w, w, y, s[0], s[1], len(x), 576, 1e-5)
        P.layernorm_backward(x, x, w, s[0], s[1], y, w.clone(), w.clone(), len(x), 576, acc=False)
        torch.cuda.synchronize()


def test_defaults_are_as_before():
    """Without the options, the model's parameters and its fused prologue are the ones it had."""
    m = SmolLM(layers=1, seq=16, rank=0, config={"vocab": 100})
    assert not any("bias" in n for n, _ in m.named_params())
    tokens = torch.randint(0, 100, (1, 16), device=DEV)
    assert torch.equal(m.hidden(tokens), m._hidden_cfops(tokens))
    with pytest.raises(ValueError, match="positions"):
        m.hidden(tokens, torch.zeros(1, 16, dtype=torch.int64, device=DEV))
    # The whole head in halves by ops.rotary is the prologue, up to f32 roundings.
    r, r2 = (SmolLM(layers=1, seq=16, rank=0, config={"vocab": 100, "rotary": o}) for o in ({}, {"dim": 64}))
    x, y = m.hidden(tokens), r.hidden(tokens)
    assert torch.equal(y, r2.hidden(tokens))
    assert bool(((x - y).abs() <= 1e-5 * (1 + x.abs())).all())


def test_refusals():
    a, b = models()
    tokens, positions, ids, z, lse = batch()
    with pytest.raises(ValueError, match="cfops"):
        b.distill(tokens, ids, z, lse)
    with pytest.raises(ValueError, match="norm"):
        SmolLM(layers=1, seq=8, rank=0, config={"norm": "batch"})
    ids[0, 1, 0] = VOCAB
    a.distill(tokens, ids, z, lse, 2.0)
    with pytest.raises(Exception, match="row 1 "):
        a.check_targets()
