"""SmolLM-135M-shaped LoRA training step with cpuforge's attention on the GPU.

This is the measurement behind "SmolLM-135M train tok/s", the second half of
the tier's metric. It follows the reference's `cpuforge bench-train`
(crates/cli/src/cmd_bench.rs:43-99):

- **Model.** A random-init SmolLM-135M shape (`smollm_135m_config`,
  cmd_bench.rs:43-50):
  - 30 layers, hidden 576, FFN 1536, 9 query / 3 KV heads of 64, vocab 49152;
  - tied embeddings, RMSNorm eps 1e-5, RoPE theta 1e4.
- **Init** (`Model::random`, crates/model/src/model.rs:282-305): weights
  N(0, 0.02), norm gains 1.
- **LoRA** (`Linear::add_lora`, crates/model/src/linear.rs:44-53):
  - rank 16, alpha 32, on q, k, v, o, gate, up, down;
  - A uniform in ±1/sqrt(in), B zero;
  - only the adapters train (`TrainSpec::LORA_ONLY`).
- **Timed step.** `grads.zero()` plus one `forward_backward` (cmd_bench.rs:78-87):
  embeddings → 30 × Layer → final norm → tied LM head → mean cross-entropy,
  then the backward. There is no optimizer step, as in the reference.
- **Batch.** The reference runs one sequence per call; this harness runs
  `batch` sequences in one device pass. tok/s = batch·seq / step time.

The attention of every layer is `cpuforge_amd.layer.layer_attention`, the
fused RoPE + attention kernels.  With `backend="cfops"` (the default) every
other op of the step also runs through libcfattn.so (include/cfops.h, via
`cpuforge_amd.autograd`): RMSNorm, the LoRA linears, the
SwiGLU gate and the LM head with its cross-entropy, whose [t, vocab] logits
are formed a chunk of rows at a time.  Only the embedding gather and the
residual adds stay torch ops.  `backend="torch"` runs those ops as plain torch
ops instead, for comparison.
"""
from __future__ import annotations

import time
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import autograd as A
from . import device as D
from .layer import LayerRope, layer_attention
from .rope import RopeCache
from .st import FormatError

SMOLLM_135M = dict(vocab=49152, d=576, ffn=1536, heads=9, kv_heads=3, head_dim=64, eps=1e-5, theta=1e4)


class LoRALinear:
    """y = x Wᵀ (+ (alpha/r) (x Aᵀ) Bᵀ with an adapter) (linear.rs:1-3, 56-69)."""

    def __init__(self, out: int, inn: int, std: float, gen, dtype, device):
        self.w = (torch.randn(out, inn, generator=gen, device=device) * std).to(dtype)
        self.a = self.b = None
        self.scale = 1.0

    def add_lora(self, rank: int, alpha: float, gen) -> None:
        """Linear::add_lora (linear.rs:44-52): A uniform in ±1/sqrt(in), B zero,
        scale alpha / rank."""
        out, inn = self.w.shape
        bound = 1.0 / inn ** 0.5
        dev, dt = self.w.device, self.w.dtype
        self.a = ((torch.rand(rank, inn, generator=gen, device=dev) * 2 - 1) * bound).to(dt).requires_grad_()
        self.b = torch.zeros(out, rank, device=dev, dtype=dt, requires_grad=True)
        self.scale = alpha / rank

    def __call__(self, x, backend="torch"):
        if backend == "cfops":
            return A.linear(x, self.w, self.a, self.b, self.scale)
        y = x @ self.w.t()
        if self.a is None:
            return y
        return y + (self.scale * (x @ self.a.t())) @ self.b.t()

    def spec(self):
        """(w, a, b, scale) for the shared-input linears."""
        return self.w, self.a, self.b, self.scale

    def named(self, prefix: str):
        """visit_linear (crates/model/src/model.rs:164-173)."""
        yield f"{prefix}.weight", self.w
        if self.a is not None:
            yield f"{prefix}.lora_A", self.a
            yield f"{prefix}.lora_B", self.b

    def params(self):
        return [self.a, self.b] if self.a is not None else []


def rmsnorm(x, w, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def rotary(x, cos, sin, positions, interleaved):
    """ops.rotary of x [B, S, H, D] in torch operations."""
    at = torch.arange(x.shape[1], device=x.device) if positions is None else positions
    c, s = cos[at].unsqueeze(-2), sin[at].unsqueeze(-2)
    half = cos.shape[1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    pair = (a * c - b * s, b * c + a * s)
    return torch.cat([torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1), rest], -1)


@dataclass
class LoraConfig:
    """crates/model/src/model.rs:45-49."""
    rank: int
    alpha: float
    targets: list


LORA_TARGETS = ("q", "k", "v", "o", "gate", "up", "down")
_LINEARS = (("q", "wq"), ("k", "wk"), ("v", "wv"), ("o", "wo"), ("gate", "gate"), ("up", "up"), ("down", "down"))


class SmolLM:
    """`rank` > 0 attaches adapters (alpha 2·rank) to every projection, as
    `cpuforge bench-train` does; `train` is the TrainSpec: "lora" trains the
    adapters only (LORA_ONLY), "full" every parameter (FULL).  `config`
    overrides entries of SMOLLM_135M (a smaller model for tests), or gives it
    another decoder's layers: norm="layer" (layer norms with a bias in the place of
    RMSNorm), rotary=dict(dim=.., interleaved=..) (the first `dim` values of
    each head turn, all by default, in halves or as pairs side by side: ops.rotary
    before the attention instead of the fused prologue, at positions of the
    caller's; the attention is over the whole row all the same), rope_scaling (a
    scaling of RopeCache)."""

    def __init__(self, layers: int = 30, seq: int = 512, rank: int = 16, dtype=torch.float32, device="cuda",
                 seed: int = 1, attn_dtype=None, backend: str = "cfops", config: dict | None = None,
                 train: str = "lora"):
        if backend not in ("cfops", "torch"):
            raise ValueError(f"unknown backend {backend!r}")
        if backend == "cfops" and dtype != torch.float32:
            raise ValueError("the cfops backend runs the reference's f32 arithmetic")
        if train not in ("lora", "full"):
            raise ValueError(f"unknown train spec {train!r}")
        c = dict(SMOLLM_135M, norm="rms", rotary=None, rope_scaling=None)
        c.update(config or {})
        if c["norm"] not in ("rms", "layer"):
            raise ValueError(f"unknown norm {c['norm']!r}")
        self.c, self.dtype, self.layers_n, self.backend, self.train = c, dtype, layers, backend, train
        self.attn_dtype = attn_dtype or dtype
        self.device = device
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        d, f, hd = c["d"], c["ffn"], c["head_dim"]
        qd, kvd = c["heads"] * hd, c["kv_heads"] * hd
        lin = lambda o, i: LoRALinear(o, i, 0.02, gen, dtype, device)  # noqa: E731
        ones = lambda: torch.ones(d, device=device, dtype=dtype)  # noqa: E731
        zeros = lambda: torch.zeros(d, device=device, dtype=dtype) if c["norm"] == "layer" else None  # noqa: E731
        self.layers = [dict(attn_norm=ones(), attn_norm_b=zeros(), wq=lin(qd, d), wk=lin(kvd, d), wv=lin(kvd, d),
                            wo=lin(d, qd), mlp_norm=ones(), mlp_norm_b=zeros(), gate=lin(f, d), up=lin(f, d),
                            down=lin(d, f)) for _ in range(layers)]
        self.embed = (torch.randn(c["vocab"], d, generator=gen, device=device) * 0.02).to(dtype)
        self.final_norm, self.final_norm_b = ones(), zeros()
        turned = (c["rotary"] or {}).get("dim", hd)
        self.rope = LayerRope(RopeCache(turned, seq, c["theta"], c["rope_scaling"]), device)
        self.attention = layer_attention  # (q_pre, k_pre, v, LayerRope) -> o
        # With ce_on_device the cfops loss leaves its value on the device
        # (no host wait: a step that can be captured in a HIP graph) and the
        # target check waits for check_targets().
        self.ce_on_device = False
        self._ce = None
        self.lora_cfg = None
        if train == "full":
            for _, p in self.named_params():
                p.requires_grad_()
        if rank:
            self.add_lora(rank, 2.0 * rank, list(LORA_TARGETS), seed)

    def add_lora(self, rank: int, alpha: float, targets, seed: int) -> None:
        """Model::add_lora (crates/model/src/model.rs:309-335): adapters on the
        named projections of every layer, initialised from `seed`."""
        for t in targets:
            if t not in LORA_TARGETS:
                raise FormatError(f"unknown LoRA target '{t}'")
        if self.lora_cfg is not None:
            raise FormatError("model already has LoRA adapters")
        gen = torch.Generator(device=self.device)
        gen.manual_seed(seed)
        for layer in self.layers:
            for short, attr in _LINEARS:
                if short in targets:
                    layer[attr].add_lora(rank, alpha, gen)
        self.lora_cfg = LoraConfig(rank, alpha, [str(t) for t in targets])

    def named_params(self):
        """visit_params order and names (crates/model/src/model.rs:179-208)."""
        yield "model.embed_tokens.weight", self.embed
        for i, layer in enumerate(self.layers):
            p = f"model.layers.{i}"
            yield f"{p}.input_layernorm.weight", layer["attn_norm"]
            if layer["attn_norm_b"] is not None:
                yield f"{p}.input_layernorm.bias", layer["attn_norm_b"]
            yield from layer["wq"].named(f"{p}.self_attn.q_proj")
            yield from layer["wk"].named(f"{p}.self_attn.k_proj")
            yield from layer["wv"].named(f"{p}.self_attn.v_proj")
            yield from layer["wo"].named(f"{p}.self_attn.o_proj")
            yield f"{p}.post_attention_layernorm.weight", layer["mlp_norm"]
            if layer["mlp_norm_b"] is not None:
                yield f"{p}.post_attention_layernorm.bias", layer["mlp_norm_b"]
            yield from layer["gate"].named(f"{p}.mlp.gate_proj")
            yield from layer["up"].named(f"{p}.mlp.up_proj")
            yield from layer["down"].named(f"{p}.mlp.down_proj")
        yield "model.norm.weight", self.final_norm
        if self.final_norm_b is not None:
            yield "model.norm.bias", self.final_norm_b

    def params(self):
        """The parameters that train (TrainSpec)."""
        return [p for _, p in self.named_params() if p.requires_grad]

    def hidden(self, tokens, positions=None):
        """The final norm's output [B, S, d].  positions [B, S] (int64; with
        config rotary): those that q and k turn by.  They do not limit the attention,
        which is causal over the row: of documents that share a row, a later one
        attends to those before it."""
        return self._hidden_cfops(tokens, positions) if self.backend == "cfops" else \
            self._hidden_torch(tokens, positions)

    def _attend(self, q, k, v, positions):
        """Layer::forward's q_pre, k_pre, v -> attn_o; with config rotary, turned by
        ops.rotary and through the attention alone."""
        if self.c["rotary"] is None:
            if positions is not None:
                raise ValueError("positions need a model with config rotary")
            return self.attention(q, k, v.to(self.attn_dtype), self.rope)
        pr, interleaved = self.rope.pr, bool(self.c["rotary"].get("interleaved"))
        if self.backend == "cfops":
            q, k = A.rotary((q, k), pr.cos, pr.sin, positions, interleaved=interleaved, dtype=self.attn_dtype)
        else:
            q, k = (rotary(x.float(), pr.cos, pr.sin, positions, interleaved).to(self.attn_dtype) for x in (q, k))
        return D.attention(q, k, v.to(self.attn_dtype))

    def _norm(self, x, w, b):
        if b is None:
            return (A.rmsnorm if self.backend == "cfops" else rmsnorm)(x, w, self.c["eps"])
        if self.backend == "cfops":
            return A.layer_norm(x, w, b, self.c["eps"])
        return F.layer_norm(x, x.shape[-1:], w, b, self.c["eps"])

    def distill(self, tokens, ids, teacher, teacher_lse=None, temperature=1.0, positions=None):
        """The rows' losses [B, S] against a teacher's top logits (A.lm_head_distill;
        ids and teacher [B, S, k], teacher_lse [B, S] or None; positions as hidden's;
        cfops backend, no host wait: check_targets() reports entries that it does not
        take)."""
        if self.backend != "cfops":
            raise ValueError("distillation needs the cfops backend")
        loss, res = A.lm_head_distill(self.hidden(tokens, positions), self.embed, ids, teacher, teacher_lse,
                                      temperature)
        self._ce = (res, None)
        return loss

    def logprobs(self, tokens, targets):
        """The targets' log-probabilities [B, S], 0 where a target is
        ops.IGNORE_INDEX (A.lm_head_logprobs; cfops backend, no host wait:
        check_targets() reports a target out of range).  What a preference or
        policy loss starts from."""
        if self.backend != "cfops":
            raise ValueError("log-probabilities need the cfops backend")
        logp, res = A.lm_head_logprobs(self.hidden(tokens), self.embed, targets)
        self._ce = (res, targets)
        return logp

    def loss(self, tokens, targets):
        if self.backend == "cfops":
            return self._loss_cfops(tokens, targets)
        logits = self.hidden(tokens) @ self.embed.t()
        return F.cross_entropy(logits.view(-1, self.c["vocab"]).float(), targets.view(-1))

    def _hidden_torch(self, tokens, positions=None):
        c = self.c
        B, S = tokens.shape
        x = self.embed[tokens]
        for layer in self.layers:
            n1 = self._norm(x, layer["attn_norm"], layer["attn_norm_b"])
            q = layer["wq"](n1).view(B, S, c["heads"], c["head_dim"])
            k = layer["wk"](n1).view(B, S, c["kv_heads"], c["head_dim"])
            v = layer["wv"](n1).view(B, S, c["kv_heads"], c["head_dim"])
            o = self._attend(q.float(), k.float(), v, positions)
            x = x + layer["wo"](o.view(B, S, -1).to(self.dtype))
            n2 = self._norm(x, layer["mlp_norm"], layer["mlp_norm_b"])
            x = x + layer["down"](F.silu(layer["gate"](n2)) * layer["up"](n2))
        return self._norm(x, self.final_norm, self.final_norm_b)

    def _hidden_cfops(self, tokens, positions=None):
        """Layer::forward (crates/model/src/layer.rs:90-143) per layer, then the
        final norm, every op but the gather and the residual adds in
        libcfattn.so."""
        c, cf = self.c, "cfops"
        B, S = tokens.shape
        x = self.embed[tokens]
        for layer in self.layers:
            n1 = self._norm(x, layer["attn_norm"], layer["attn_norm_b"])
            q, k, v = A.shared_input_linears(n1, [layer[n].spec() for n in ("wq", "wk", "wv")])
            q = q.view(B, S, c["heads"], c["head_dim"])
            k = k.view(B, S, c["kv_heads"], c["head_dim"])
            v = v.view(B, S, c["kv_heads"], c["head_dim"])
            o = self._attend(q, k, v, positions)
            x = x + layer["wo"](o.view(B, S, -1), cf)
            n2 = self._norm(x, layer["mlp_norm"], layer["mlp_norm_b"])
            g, u = A.shared_input_linears(n2, [layer[n].spec() for n in ("gate", "up")])
            x = x + layer["down"](A.silu_mul(g, u), cf)
        return self._norm(x, self.final_norm, self.final_norm_b)

    def _loss_cfops(self, tokens, targets):
        """The tied LM head with its loss (model.rs:436-442)."""
        hn = self._hidden_cfops(tokens)
        if self.ce_on_device:
            loss, res = A.lm_head_ce_dev(hn, self.embed, targets)
            self._ce = (res, targets)
            return loss
        return A.lm_head_ce(hn, self.embed, targets)

    def check_targets(self) -> None:
        """Raises, as the loss would have, if the last device-side loss met
        a target out of range (waits for it)."""
        if self._ce is not None:
            from .ops import ce_check, distill_check
            res, targets = self._ce
            if targets is None:
                distill_check(res)
            else:
                ce_check(res, targets, self.c["vocab"])


def capture_step(model: SmolLM, tokens, targets, warmup: int = 2):
    """The training step (every trained parameter's .grad reset, forward,
    loss, backward) captured in a HIP graph: `warmup` eager steps on a side
    stream (the capture recipe: the library's scratch and
    torch's allocations are made there), then the capture.  Returns the graph
    and the loss tensor its replays write; each replay leaves the step's
    gradients in the parameters' .grad.  Needs the cfops backend with
    model.ce_on_device, so that no op waits for the host."""
    if model.backend != "cfops" or not model.ce_on_device:
        raise ValueError("graph capture needs the cfops backend with ce_on_device")
    params = model.params()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(warmup):
            for p_ in params:
                p_.grad = None
            loss = model.loss(tokens, targets)
            loss.backward()
            del loss
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    model.check_targets()
    for p_ in params:
        p_.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static_loss = model.loss(tokens, targets)
        static_loss.backward()
    return graph, static_loss


def train_tok_s(batch: int = 8, seq: int = 512, layers: int = 30, rank: int = 16, steps: int = 3,
                dtype=torch.float32, attn_dtype=None, device="cuda", backend: str = "cfops",
                warmup: int = 3, graph: bool = False) -> dict:
    """Build the model, run `warmup` untimed steps (the first allocates the
    library's scratch; the clock settles over the next ones),
    then time `steps` forward+backward passes; returns tok/s and the step
    time.  With `graph` (cfops backend) the step is captured in a HIP graph
    after the warm-up steps and the timed steps are its replays: the same
    kernels in the same order, without the host's launch work between
    them."""
    model = SmolLM(layers, seq, rank, dtype, device, attn_dtype=attn_dtype, backend=backend)
    gen = torch.Generator(device=device)
    gen.manual_seed(7)
    tokens = torch.randint(0, model.c["vocab"], (batch, seq), generator=gen, device=device)
    targets = torch.randint(0, model.c["vocab"], (batch, seq), generator=gen, device=device)
    params = model.params()

    def step():
        for p_ in params:
            p_.grad = None
        loss = model.loss(tokens, targets)
        loss.backward()
        return loss

    loss0 = step().item()
    out = {}
    if graph:
        model.ce_on_device = True
        g, static_loss = capture_step(model, tokens, targets, max(warmup - 1, 1))
        g.replay()
        torch.cuda.synchronize()
        model.check_targets()
        out["graph_first_loss"] = static_loss.item()
        run = g.replay
    else:
        for _ in range(warmup - 1):
            step()
        run = step
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        run()
    torch.cuda.synchronize()
    per = (time.perf_counter() - t0) / steps
    if graph:
        model.check_targets()
    return {"value": batch * seq / per, "unit": "tok/s", "ms_per_step": per * 1e3, "batch": batch, "seq": seq,
            "layers": layers, "lora_rank": rank, "dtype": str(dtype).replace("torch.", ""),
            "attn_dtype": str(attn_dtype or dtype).replace("torch.", ""), "steps": steps, "warmup": warmup,
            "first_loss": loss0, "backend": backend, "graph": graph, **out}
