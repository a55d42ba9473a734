"""The preference- and policy-training operators as timed and compared cases.

A finetuning step on preferences or rewards runs the hidden states through the
LM head into the targets' log-probabilities (`ops.lm_head_logprobs`, and
`autograd.lm_head_logprobs` with its backward), those into a preference loss
over pairs of sequences (`ops.preference_loss`) or a clipped policy loss with a
KL term (`ops.policy_loss`), and the gradients into an AdamW step whose moments
are held in 8 bits (`ops.adamw8_update_multi`).

`listed()` names the cases, `draw(rng)` gives another one of the same ranges;
`prepare` / `run` / `work` / `exact` describe one case.  With `own` false, `run`
computes the same in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
IGNORE = -100
BLOCK = 256  # values of an 8-bit state that share a power of two
SMALL = 4096  # tensors with fewer values keep 32-bit states
# One optimizer step some way into training.
STEP, LR, BETA1, BETA2, EPS, DECAY = 11, 1e-4, 0.9, 0.999, 1e-8, 0.01
# Loss settings in common use.
BETA, SMOOTHING, MARGIN = 0.1, 0.1, 0.05
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04

# --------------------------------------------------------------------- cases


def listed():
    return [
        # Scoring the next token of one sequence at SmolLM-135M's head.
        dict(name="logp_token", kind="logp", tokens=1, d=576, vocab=49152, seq=1, prompt=0),
        # The reference model's pass of a preference batch: eight sequences of
        # 512 tokens of which half are prompts.
        dict(name="logp_reference", kind="logp", tokens=4096, d=576, vocab=49152, seq=512, prompt=256),
        # The same at Llama-3.2-1B's head, an odd number of tokens.
        dict(name="logp_wide", kind="logp", tokens=1001, d=2048, vocab=128256, seq=143, prompt=13),
        # The trained model's pass with a frozen head (adapters train): the
        # log-probabilities and the hidden states' gradients.
        dict(name="train_frozen_head", kind="train", tokens=4096, d=576, vocab=49152, seq=512, prompt=51,
             head_grad=False),
        # The head trains too; nothing is a multiple of a tile.
        dict(name="train_full_head", kind="train", tokens=999, d=500, vocab=50001, seq=111, prompt=20,
             head_grad=True),
        # The loss of one small preference batch: latency.
        dict(name="preference_small", kind="preference", pairs=4, longest=90, form="sigmoid", length_mean=False,
             reference=True),
        # A large one of ragged lengths, means over the tokens and no reference.
        dict(name="preference_large", kind="preference", pairs=400, longest=2048, form="sigmoid", length_mean=True,
             reference=False),
        # A small group of rollouts, one advantage each.
        dict(name="policy_small", kind="policy", seqs=8, longest=120, per_token=False, reference=True,
             reduction="sequence"),
        # A large batch of rollouts with advantages by token.
        dict(name="policy_large", kind="policy", seqs=1024, longest=1800, per_token=True, reference=True,
             reduction="token"),
        # An optimizer step over SmolLM-135M's adapters of rank 8, most of them
        # small.
        dict(name="adamw8_adapters", kind="adamw8", model="adapters", layers=30, rank=8, shift=0),
        # Over all of its parameters: the embedding, the projections and the
        # norms (whose states stay in 32 bits).
        dict(name="adamw8_full", kind="adamw8", model="full", layers=30, rank=0, shift=0),
        # Over tensors of odd sizes that start off a 16-byte boundary.
        dict(name="adamw8_odd", kind="adamw8", model="odd", layers=9, rank=0, shift=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("logp", "logp", "train", "train", "preference", "policy", "adamw8"))
    if kind in ("logp", "train"):
        d = rng.choice((576, 576, 500, 1024, 2048, 129))
        vocab = rng.choice((49152, 49152, 32000, 50001, 128256, 1000))
        most = int((5.0e11 if kind == "logp" else 2.5e11) / (2 * d * vocab))
        tokens = _log(rng, 1 if kind == "logp" else 16, max(16, min(4096, most)))
        seq = min(tokens, _log(rng, 16, 512))
        c = dict(kind=kind, tokens=tokens, d=d, vocab=vocab, seq=seq, prompt=rng.randint(0, seq // 2))
        if kind == "train":
            c["head_grad"] = rng.random() < 0.4 and tokens * d * vocab < 6e10
        return c
    if kind == "preference":
        pairs = _log(rng, 1, 400)
        return dict(kind=kind, pairs=pairs, longest=_log(rng, 20, min(32768, 800000 // pairs)),
                    form=rng.choice(("sigmoid", "sigmoid", "hinge", "squared")), length_mean=rng.random() < 0.5,
                    reference=rng.random() < 0.7)
    if kind == "policy":
        seqs = _log(rng, 1, 1024)
        return dict(kind=kind, seqs=seqs, longest=_log(rng, 20, min(65536, 1800000 // seqs)),
                    per_token=rng.random() < 0.5, reference=rng.random() < 0.6,
                    reduction=rng.choice(("token", "sequence")))
    model = rng.choice(("adapters", "full", "odd", "odd"))
    if model == "adapters":
        return dict(kind=kind, model=model, layers=rng.randint(2, 30), rank=rng.choice((4, 8, 10, 12)), shift=0)
    if model == "full":
        return dict(kind=kind, model=model, layers=rng.randint(1, 29), rank=0, shift=0)
    return dict(kind=kind, model=model, layers=rng.randint(1, 24), rank=0, shift=rng.choice((0, 0, 1, 3)))


# ------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def _scored(tokens, seq, prompt):
    """Rows whose next token counts: not a prompt's."""
    return np.arange(tokens) % seq >= prompt


def _head_inputs(case, seed):
    g = _gen(seed)
    t, d, vocab = case["tokens"], case["d"], case["vocab"]
    s = dict(hn=_randn(g, t, d), head=_randn(g, vocab, d, std=0.02),
             targets=torch.randint(0, vocab, (t,), generator=g, device=DEV))
    s["targets"][torch.from_numpy(~_scored(t, case["seq"], case["prompt"])).to(DEV)] = IGNORE
    # A gradient per row, as a preference loss gives it: one value a sequence.
    s["dlogp"] = (_randn(g, (t + case["seq"] - 1) // case["seq"], std=0.02)
                  .repeat_interleave(case["seq"])[:t].contiguous())
    return s


def _lengths(count, longest):
    """Ragged lengths in [longest / 4, longest], the same for every seed."""
    r = np.random.RandomState(count * 7919 + longest)
    return r.randint(max(1, longest // 4), longest + 1, size=count)


TAIL = 5  # rows behind the last sequence, which stay as they were


def _sequence_inputs(case, seed):
    """Log-probabilities of ragged sequences whose first tenth is a prompt."""
    g = _gen(seed)
    count = 2 * case["pairs"] if case["kind"] == "preference" else case["seqs"]
    lengths = _lengths(count, case["longest"])
    off = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    rows = int(off[-1]) + TAIL
    offsets = torch.from_numpy(off).to(DEV)
    at = torch.arange(rows, device=DEV)
    seq = (torch.searchsorted(offsets, at, right=True) - 1).clamp(max=count - 1)
    targets = torch.randint(0, 49152, (rows,), generator=g, device=DEV)
    prompt = torch.from_numpy(lengths // 10).to(DEV)
    targets[at - offsets[seq] < prompt[seq]] = IGNORE
    ref = -torch.rand(rows, generator=g, device=DEV).mul_(6.0)
    logp = ref + _randn(g, rows, std=0.1)
    s = dict(offsets=offsets, targets=targets, logp=logp, ref=ref if case["reference"] else None, rows=rows,
             count=count, dlogp=torch.zeros(rows, device=DEV))
    if case["kind"] == "policy":
        s["old"] = logp + _randn(g, rows, std=0.15)
        s["adv"] = _randn(g, rows if case["per_token"] else count)
    return s


def _adamw_sizes(case):
    """(values, weight decay) of the tensors of a step."""
    d, f, kv, vocab = 576, 1536, 192, 49152
    linears = ((d, d), (kv, d), (kv, d), (d, d), (f, d), (f, d), (d, f))
    if case["model"] == "adapters":
        r = case["rank"]
        return [(n, DECAY) for _ in range(case["layers"]) for o, i in linears for n in (r * i, o * r)]
    if case["model"] == "full":
        layer = [(o * i, DECAY) for o, i in linears] + [(d, 0.0), (d, 0.0)]
        return [(vocab * d, DECAY)] + layer * case["layers"] + [(d, 0.0)]
    odd = (1, 255, 4099, 1000003, 65537, 257, 300001, 4095, 8191)
    return [(odd[i % len(odd)] + 2 * (i // len(odd)), DECAY * (i % 3)) for i in range(case["layers"])]


def _extents(sizes):
    """Each tensor's first value in buffers that start every tensor on a block."""
    padded = [-(-n // BLOCK) * BLOCK for n, _ in sizes]
    return np.concatenate([[0], np.cumsum(padded)]).astype(np.int64)


def _exponents(a):
    """e of each magnitude's binade [2^e, 2^(e+1)); -127 for 0."""
    return torch.where(a > 0, torch.frexp(a)[1] - 1, -127).clamp(-127, 127)


def _dither(i, step):
    """17 random bits for each state of value i of a tensor in a step, as whole
    numbers: the value's rounding threshold."""
    def mix(x):
        x = (x ^ (x >> 16)) * 0xA511E9B3 & 0xFFFFFFFF
        x = (x ^ (x >> 15)) * 0x63D83595 & 0xFFFFFFFF
        return x ^ (x >> 16)
    key = mix(torch.full((), (step * 0x9E3779B1 + 0x7F4A7C15) & 0xFFFFFFFF, dtype=torch.int64, device=DEV))
    h = mix((i + key) & 0xFFFFFFFF)
    return h & 0x1FFFF, h >> 15


def _held(a, least, threshold):
    """Blocks [n, 256] of 64-bit magnitudes as 8 bits hold them: three mantissa
    bits behind the leading one down to the binade 2^(E + least), and steps of
    that binade's below it, E the block's power of two: its largest value is in
    (2^E, 2^(E+1)].  A value between two steps goes up where the fraction of
    the step that it has passed and its threshold make a whole one, so that
    the mean of many roundings is the value: a moment that moves by less than a
    step a time would never move else."""
    big = a.amax(1, keepdim=True)
    # (Up to 2^-20 above a power of two counts as that power.)
    top = _exponents(big * (1 - 2.0 ** -20))
    step = torch.exp2((torch.maximum(_exponents(a), top + least) - 3).to(a.dtype))
    return torch.floor(a / step + threshold * 2.0 ** -17) * step, top


def _held_m(m, threshold):
    return torch.copysign(_held(m.abs(), -13, threshold)[0], m)


def _held_v(v, threshold):
    """(A second moment that is not zero is not held as zero.)"""
    h, top = _held(v, -29, threshold)
    return torch.where(v > 0, torch.maximum(h, torch.exp2((top - 32).to(v.dtype))), h)


def _adamw_inputs(case, seed):
    """Parameters with a gradient each and the moments some steps into
    training, each kind side by side in one buffer."""
    g = _gen(seed)
    sizes = _adamw_sizes(case)
    ext = _extents(sizes)
    total = int(ext[-1])
    blocks = np.diff(ext) // BLOCK
    lens = torch.tensor([n for n, _ in sizes], device=DEV)
    which = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.from_numpy(blocks).to(DEV))
    at = torch.arange(total, device=DEV).view(-1, BLOCK)
    index = at - torch.from_numpy(ext[:-1].copy()).to(DEV)[which][:, None]
    live = index < lens[which][:, None]
    in8 = (lens >= SMALL)[which][:, None]
    decay = torch.tensor([w for _, w in sizes], device=DEV)[which][:, None]
    # (p and g start `shift` values off the block's boundary.)
    sh = case["shift"]
    whole = {n: torch.zeros(total + sh, device=DEV) for n in ("p", "g")}
    flat = {n: t[sh:] for n, t in whole.items()}
    flat["p"].copy_(torch.where(live, _randn(g, total // BLOCK, BLOCK, std=0.02), 0.0).view(-1))
    # Gradients of blocks differ in size, as those of rows of a weight do.
    size = torch.exp(_randn(g, total // BLOCK, 1)) * 1e-3
    flat["g"].copy_(torch.where(live, _randn(g, total // BLOCK, BLOCK) * size, 0.0).view(-1))
    m = torch.where(live, _randn(g, total // BLOCK, BLOCK) * size * 0.3, 0.0).double()
    v = torch.where(live, (_randn(g, total // BLOCK, BLOCK) * size * 0.7).square(), 0.0).double()
    flat["m"] = torch.where(in8, _held_m(m, 1 << 16), m).float().view(-1)
    flat["v"] = torch.where(in8, _held_v(v, 1 << 16), v).float().view(-1)
    return dict(flat=flat, sizes=sizes, ext=ext, in8=in8, decay=decay, index=index)


def _adamw_table(s):
    """The library's view of the same buffers: a table of tensors, those of
    SMALL values and more with states packed to 8 bits."""
    from cpuforge_amd import ops as P
    f = s["flat"]
    cut = [{k: f[k][int(o):int(o) + n] for k in "pgmv"} for o, (n, _) in zip(s["ext"], s["sizes"])]
    for c, (n, w) in zip(cut, s["sizes"]):
        c["weight_decay"] = w
        if n >= SMALL:
            c["state8"] = P.adamw8_state(n, DEV)
    table = P.Adamw8Tensors(cut)
    P.adamw8_pack_multi(table)
    return table


def prepare(case, seed):
    kind = case["kind"]
    if kind in ("logp", "train"):
        s = _head_inputs(case, seed)
        t = case["tokens"]
        if kind == "logp":
            s["logp"], s["lse"] = torch.empty(t, device=DEV), torch.empty(t, device=DEV)
            s["result"] = torch.zeros(3, dtype=torch.int32, device=DEV)
        else:
            s["hn"].requires_grad_()
            s["head"].requires_grad_(case["head_grad"])
        return dict(case=case, **s)
    if kind in ("preference", "policy"):
        s = _sequence_inputs(case, seed)
        if kind == "preference":
            s["rewards"] = torch.empty(s["count"], device=DEV)
        s["result"] = torch.zeros(8, dtype=torch.int32, device=DEV)
        return dict(case=case, **s)
    s = _adamw_inputs(case, seed)
    if own:
        s["table"] = _adamw_table(s)
    return dict(case=case, **s)


# -------------------------------------------------------------- plain forms


def _plain_logp(hn, head, targets):
    """(logp, lse, scored rows, their logits)."""
    idx = torch.nonzero(targets != IGNORE).view(-1)
    logits = hn[idx] @ head.T
    top = logits.amax(1, keepdim=True)
    l_ = (top + (logits - top).exp().sum(1, keepdim=True).log()).view(-1)
    logp, lse = torch.zeros_like(targets, dtype=torch.float32), torch.zeros_like(targets, dtype=torch.float32)
    lse[idx] = l_
    logp[idx] = logits.gather(1, targets[idx][:, None]).view(-1) - l_
    return logp, lse, idx, logits


def _plain_train(s):
    hn, head, targets = s["hn"].detach(), s["head"].detach(), s["targets"]
    logp, lse, idx, logits = _plain_logp(hn, head, targets)
    g = s["dlogp"][idx][:, None]
    dl = (logits - lse[idx][:, None]).exp() * -g
    dl.scatter_add_(1, targets[idx][:, None], g)
    dhn = torch.zeros_like(hn)
    dhn[idx] = dl @ head
    return (logp, dhn, dl.T @ hn[idx]) if s["case"]["head_grad"] else (logp, dhn)


def _by_sequence(s):
    """(sequence of each row of one, whether it is scored), of the rows of sequences."""
    rows = s["rows"] - TAIL
    at = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(s["offsets"], at, right=True) - 1
    return rows, seq, s["targets"][:rows] != IGNORE


def _sums(x, seq, count):
    return torch.zeros(count, dtype=torch.float64, device=DEV).index_add_(0, seq, x)


def _plain_preference(s):
    """Sums in 64 bits: long sequences' are, and the pairs' differences cancel."""
    c = s["case"]
    rows, seq, scored = _by_sequence(s)
    x = s["logp"][:rows].double()
    if s["ref"] is not None:
        x = x - s["ref"][:rows].double()
    total = _sums(torch.where(scored, x, 0.0), seq, s["count"])
    n = _sums(scored.double(), seq, s["count"])
    per = 1.0 / n.clamp(min=1.0) if c["length_mean"] else torch.ones_like(n)
    rewards = BETA * total * per
    chosen, rejected = rewards.view(-1, 2).unbind(1)
    z = chosen - rejected - MARGIN
    if c["form"] == "sigmoid":
        up, down = torch.exp(-z.abs()), 1.0 / (1.0 + torch.exp(-z.abs()))
        soft = torch.log1p(up)
        loss = (1 - SMOOTHING) * (soft + (-z).clamp(min=0)) + SMOOTHING * (soft + z.clamp(min=0))
        sig = torch.where(z >= 0, down, up * down)
        dz = (1 - SMOOTHING) * (sig - 1) + SMOOTHING * sig
    elif c["form"] == "hinge":
        loss, dz = (1 - z).clamp(min=0), torch.where(z < 1, -1.0, 0.0).double()
    else:
        loss, dz = (z - 0.5) ** 2, 2 * (z - 0.5)
    sign = torch.stack([dz, -dz], 1).view(-1) * BETA / c["pairs"] * per
    s["dlogp"][:rows] = torch.where(scored, sign[seq], 0.0).float()
    return dict(loss=loss.mean().float(), accuracy=(chosen > rejected).double().mean().float(),
                margin=(chosen - rejected).mean().float(), rewards=rewards.float(), dlogp=s["dlogp"])


def _plain_policy(s):
    """In 64 bits: whether a ratio passes its border decides a whole gradient."""
    c = s["case"]
    rows, seq, scored = _by_sequence(s)
    n = _sums(scored.double(), seq, s["count"])
    if c["reduction"] == "token":
        w = (1.0 / n.sum().clamp(min=1.0)).expand(rows)
    else:
        w = (1.0 / (n.clamp(min=1.0) * (n > 0).sum().clamp(min=1)))[seq]
    w = torch.where(scored, w, 0.0)
    lp = s["logp"][:rows].double()
    adv = (s["adv"][:rows] if c["per_token"] else s["adv"][seq]).double()
    ratio = (lp - s["old"][:rows].double()).exp()
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    cut = ratio * adv > clipped * adv
    loss, dlp = -torch.minimum(ratio * adv, clipped * adv), torch.where(cut, 0.0, -ratio * adv)
    kl = torch.zeros((), dtype=torch.float64, device=DEV)
    if s["ref"] is not None:
        x = s["ref"][:rows].double() - lp
        k3 = torch.expm1(x) - x
        kl = (k3 * w).sum()
        loss, dlp = loss + KL_COEF * k3, dlp - KL_COEF * torch.expm1(x)
    s["dlogp"][:rows] = (dlp * w).float()
    clip = (cut & scored).double().sum() / n.sum().clamp(min=1.0)
    return dict(loss=(loss * w).sum().float(), kl=kl.float(), clipped=clip.float(), dlogp=s["dlogp"])


def _plain_adamw(s):
    """The moments in 64 bits: a rounding to 8 goes by what lies below 32."""
    f = s["flat"]
    p, g, m, v = (f[k].view(-1, BLOCK) for k in "pgmv")
    b1, b2 = np.float32(BETA1), np.float32(BETA2)
    c1, c2 = 1.0 / (1.0 - float(b1) ** STEP), 1.0 / math.sqrt(1.0 - float(b2) ** STEP)
    g64 = g.double()
    m2 = m.double() * float(b1) + g64 * float(np.float32(1) - b1)
    v2 = v.double() * float(b2) + (g64 * float(np.float32(1) - b2)) * g64
    upd = (m2.float() * c1) / (v2.float().sqrt() * c2 + EPS) + s["decay"] * p
    p.sub_(upd * LR)
    tm, tv = _dither(s["index"], STEP)
    m.copy_(torch.where(s["in8"], _held_m(m2, tm), m2))
    v.copy_(torch.where(s["in8"], _held_v(v2, tv), v2))
    return {k: f[k] for k in "pmv"}


# ----------------------------------------------------------------- one pass


def _own(s):
    from cpuforge_amd import autograd as A
    from cpuforge_amd import ops as P
    c = s["case"]
    if c["kind"] == "logp":
        P.lm_head_logprobs(s["hn"], s["head"], s["targets"], c["tokens"], c["d"], c["vocab"], s["logp"], s["lse"],
                           s["result"])
        return s["logp"], s["lse"]
    if c["kind"] == "train":
        logp, _ = A.lm_head_logprobs(s["hn"], s["head"], s["targets"])
        inputs = [s["hn"]] + ([s["head"]] if c["head_grad"] else [])
        return (logp.detach(), *torch.autograd.grad(logp, inputs, s["dlogp"]))
    if c["kind"] == "preference":
        P.preference_loss(s["logp"], s["ref"], s["targets"], s["offsets"], s["dlogp"], s["rewards"], s["result"],
                          beta=BETA, form=c["form"], margin=MARGIN,
                          label_smoothing=SMOOTHING if c["form"] == "sigmoid" else 0.0, length_mean=c["length_mean"])
        r = P.preference_result(s["result"])
        return dict(loss=r.loss, accuracy=r.accuracy, margin=r.margin, rewards=s["rewards"], dlogp=s["dlogp"])
    if c["kind"] == "policy":
        P.policy_loss(s["logp"], s["old"], s["ref"], s["adv"], s["targets"], s["offsets"], s["dlogp"], s["result"],
                      clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF, reduction=c["reduction"])
        r = P.policy_result(s["result"])
        return dict(loss=r.loss, kl=r.kl, clipped=r.clipped, dlogp=s["dlogp"])
    P.adamw8_update_multi(s["table"], STEP, LR, BETA1, BETA2, EPS)
    # The moments as the values they stand for.
    P.adamw8_unpack_multi(s["table"])
    return {k: s["flat"][k] for k in "pmv"}


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "logp":
        return _plain_logp(s["hn"], s["head"], s["targets"])[:2]
    if kind == "train":
        return _plain_train(s)
    if kind == "preference":
        return _plain_preference(s)
    return _plain_policy(s) if kind == "policy" else _plain_adamw(s)


def work(case):
    """Each input read once, each output written once."""
    kind = case["kind"]
    if kind in ("logp", "train"):
        t, d, vocab = case["tokens"], case["d"], case["vocab"]
        n = int(_scored(t, case["seq"], case["prompt"]).sum())
        bytes_, flops = 4 * (n * d + vocab * d) + 16 * t, 2.0 * n * d * vocab
        if kind == "train":
            bytes_ += 4 * t * d + 4 * t + (4 * vocab * d if case["head_grad"] else 0)
            flops *= 3 if case["head_grad"] else 2
        return dict(bytes=bytes_, flops=flops)
    if kind == "preference":
        rows = int(_lengths(2 * case["pairs"], case["longest"]).sum())
        return dict(bytes=rows * (16 + 4 * case["reference"]) + 24 * case["pairs"] + 8, flops=4.0 * rows)
    if kind == "policy":
        rows = int(_lengths(case["seqs"], case["longest"]).sum())
        return dict(bytes=rows * (20 + 4 * case["reference"] + 4 * case["per_token"]) + 12 * case["seqs"],
                    flops=40.0 * rows)
    sizes = _adamw_sizes(case)
    # p read and written, g read, two states of a byte read and written and
    # given as values (4 bytes each way where they are held in 32 bits).
    return dict(bytes=sum(n * ((12 + 4 + 8) if n >= SMALL else (12 + 16)) for n, _ in sizes),
                flops=20.0 * sum(n for n, _ in sizes))


# -------------------------------------------------------------------- exact


def _exact_head(case, s):
    hn, head, t64 = s["hn"].detach().double(), s["head"].detach().double(), s["targets"]
    n = t64.numel()
    logp, lse = torch.zeros(n, dtype=torch.float64, device=DEV), torch.zeros(n, dtype=torch.float64, device=DEV)
    train = case["kind"] == "train"
    dhn = torch.zeros_like(hn) if train else None
    dhead = torch.zeros_like(head) if train and case["head_grad"] else None
    keep = t64 >= 0
    for a in range(0, n, 512):
        k = keep[a:a + 512]
        if not bool(k.any()):
            continue
        x = hn[a:a + 512] @ head.T
        whole = torch.logsumexp(x, 1)
        tgt = t64[a:a + 512].clamp(min=0)[:, None]
        logp[a:a + 512] = torch.where(k, x.gather(1, tgt)[:, 0] - whole, 0.0)
        lse[a:a + 512] = torch.where(k, whole, 0.0)
        if train:
            g = torch.where(k, s["dlogp"][a:a + 512].double(), 0.0)
            one = torch.zeros_like(x).scatter_(1, tgt, 1.0)
            dx = (one - torch.softmax(x, 1)) * g[:, None]
            dhn[a:a + 512] = dx @ head
            if dhead is not None:
                dhead += dx.T @ hn[a:a + 512]
    if not train:
        return logp, lse
    return (logp, dhn) if dhead is None else (logp, dhn, dhead)


def _host(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _exact_preference(case, s):
    logp, ref, off = _host(s["logp"]), _host(s["ref"]), s["offsets"].cpu().numpy()
    use = s["targets"].cpu().numpy() >= 0
    d = logp - (0.0 if ref is None else ref)
    d = np.where(use, d, 0.0)
    reward, share = np.zeros(s["count"]), np.zeros(s["count"])
    for i in range(s["count"]):
        part = slice(off[i], off[i + 1])
        cnt = int(use[part].sum())
        share[i] = BETA / max(cnt, 1) if case["length_mean"] else BETA
        reward[i] = math.fsum(d[part]) * share[i]
    diff = reward[0::2] - reward[1::2]
    z = diff - MARGIN
    if case["form"] == "sigmoid":
        loss = (1 - SMOOTHING) * np.logaddexp(0, -z) + SMOOTHING * np.logaddexp(0, z)
        slope = 1 / (1 + np.exp(-z)) - (1 - SMOOTHING)
    elif case["form"] == "hinge":
        loss, slope = np.maximum(0, 1 - z), -(z < 1).astype(float)
    else:
        loss, slope = (z - 0.5) ** 2, 2 * z - 1
    out = np.zeros(s["rows"])
    for i in range(s["count"]):
        part = slice(off[i], off[i + 1])
        out[part] = use[part] * (slope[i // 2] * (1 - 2 * (i % 2)) * share[i] / case["pairs"])
    return dict(loss=loss.mean(), accuracy=float(np.mean(diff > 0)), margin=diff.mean(), rewards=reward, dlogp=out)


def _exact_policy(case, s):
    logp, old, ref, adv = (_host(s[k]) for k in ("logp", "old", "ref", "adv"))
    use, off = s["targets"].cpu().numpy() >= 0, s["offsets"].cpu().numpy()
    counts = np.array([int(use[off[i]:off[i + 1]].sum()) for i in range(s["count"])])
    out, loss, kl, cuts = np.zeros(s["rows"]), [], [], 0
    for i in range(s["count"]):
        part = slice(off[i], off[i + 1])
        if counts[i] == 0:
            continue
        weight = 1 / counts.sum() if case["reduction"] == "token" else 1 / (counts[i] * (counts > 0).sum())
        a = adv[part] if case["per_token"] else np.full(off[i + 1] - off[i], adv[i])
        r = np.exp(logp[part] - old[part])
        # Past the border on the side that the advantage pushes to.
        past = ((a > 0) & (r > 1 + CLIP_HIGH)) | ((a < 0) & (r < 1 - CLIP_LOW))
        held = np.where(a > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)
        l_, slope = -np.where(past, held, r) * a, np.where(past, 0.0, -r * a)
        if ref is not None:
            q = ref[part] - logp[part]
            k = np.expm1(q) - q
            l_, slope = l_ + KL_COEF * k, slope - KL_COEF * np.expm1(q)
            kl.append(weight * math.fsum(k[use[part]]))
        loss.append(weight * math.fsum(l_[use[part]]))
        cuts += int((past & use[part]).sum())
        out[part] = np.where(use[part], slope * weight, 0.0)
    return dict(loss=math.fsum(loss), kl=math.fsum(kl), clipped=cuts / max(1, counts.sum()), dlogp=out)


def _grid(a, floor, key):
    """Magnitudes [n, 256] on the steps that 8 bits have: eighths of a power of
    two, the smallest `floor` below the block's; `key` in [0, 1) decides between
    the two nearest."""
    big = a.amax(1, keepdim=True).clamp(min=2.0 ** -200)
    lead = torch.floor(torch.log2(big))
    lead = torch.where(big * torch.exp2(-lead) < 1, lead - 1, lead)
    lead = torch.where(big * torch.exp2(-lead) >= 2, lead + 1, lead)
    lead = torch.where(big * torch.exp2(-lead) < 1 + 2.0 ** -20, lead - 1, lead).clamp(min=-127)
    least = torch.exp2(lead - floor)
    low = torch.exp2(torch.floor(torch.log2(torch.maximum(a, least))))
    low = torch.where(low > torch.maximum(a, least), low / 2, low) / 8
    whole = torch.floor(a / low)
    return (whole + ((a / low - whole) >= 1 - key)) * low, least / 8


def _exact_adamw(case, s):
    """In slices of blocks."""
    f = s["flat"]
    out = {k: torch.empty(f[k].numel(), dtype=torch.float64, device=DEV) for k in "pmv"}
    n, part = f["p"].numel() // BLOCK, 1 << 16
    b1, b2 = float(np.float32(BETA1)), float(np.float32(BETA2))

    def scramble(x):
        for s_, k in ((16, 0xA511E9B3), (15, 0x63D83595)):
            x = torch.bitwise_xor(x, x >> s_) * k % 2 ** 32
        return torch.bitwise_xor(x, x >> 16)

    start = int(scramble(torch.tensor((STEP * 0x9E3779B1 + 0x7F4A7C15) % 2 ** 32)))
    for a in range(0, n, part):
        b = min(n, a + part)
        at = slice(a * BLOCK, b * BLOCK)
        p, g, m, v = (f[k][at].double().view(-1, BLOCK) for k in "pgmv")
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        mh, vh = m / (1 - b1 ** STEP), v / (1 - b2 ** STEP)
        out["p"][at] = (p - LR * (mh / (vh.sqrt() + EPS) + s["decay"][a:b].double() * p)).view(-1)
        bits = scramble((s["index"][a:b] + start) % 2 ** 32)
        q, _ = _grid(m.abs(), 13, (bits % 2 ** 17) / 2.0 ** 17)
        r, unit = _grid(v, 29, (bits // 2 ** 15) / 2.0 ** 17)
        r = torch.where((v > 0) & (r == 0), unit.expand_as(r), r)
        small = ~s["in8"][a:b]
        out["m"][at] = torch.where(small, m, q * m.sign()).view(-1)
        out["v"][at] = torch.where(small, v, r).view(-1)
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind in ("logp", "train"):
        return _exact_head(case, _head_inputs(case, seed))
    if kind in ("preference", "policy"):
        s = _sequence_inputs(case, seed)
        return _exact_preference(case, s) if kind == "preference" else _exact_policy(case, s)
    return _exact_adamw(case, _adamw_inputs(case, seed))
