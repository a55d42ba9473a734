"""AdamW over a model's device-resident parameters (crates/train/src/optim.rs).

`AdamW` keeps the reference struct's fields (beta1, beta2, eps,
weight_decay, `step` = optimizer steps taken, `state` = first and second
moments keyed by parameter name, optim.rs:32-41).  Its `update` is the
reference's `AdamW::step` (optim.rs:48-61): the count goes up by one, and every
parameter that has a gradient gets `adamw_update` (cfops_adamw_update, bitwise
the reference's f32 arithmetic) with no weight decay for the norm gains.  (The
method is not called `step` because Python cannot hold a field and a method of
one name.)

With state_bits=8 (no reference counterpart) the moments of every parameter of
at least SMALL values are held in 8 bits (`State8`; cfops_adamw8_update_multi):
two bytes and a 128th of state a value instead of eight.

A model here is any object whose `named_params()` yields (name, tensor) in
`visit_params` order (crates/model/src/model.rs:179-208); a parameter has a
gradient when it requires one, as a non-empty `Grads` entry does in the
reference (TrainSpec decides both).
"""
from __future__ import annotations

import torch

from . import ops as P

#: Parameters with fewer values keep 32-bit states: norm gains and small
#: adapters, whose states are no part of the memory and whose steps count most.
SMALL = 4096


class State8:
    """Both moments of one parameter in 8 bits."""

    def __init__(self, p: torch.Tensor):
        self.shape = p.shape
        self.buf = P.adamw8_state(p.numel(), p.device)

    @staticmethod
    def pack(m: torch.Tensor, v: torch.Tensor) -> "State8":
        s = State8(m)
        P.adamw8_pack_multi([dict(m=m.contiguous(), v=v.contiguous(), state8=s.buf)])
        return s

    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(m, v) as f32 tensors, which pack to the same state."""
        m, v = (torch.empty(self.shape, device=self.buf.device, dtype=torch.float32) for _ in range(2))
        P.adamw8_unpack_multi([dict(m=m, v=v, state8=self.buf)])
        return m, v


class AdamW:
    def __init__(self, beta1: float, beta2: float, eps: float, weight_decay: float, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.beta1, self.beta2, self.eps, self.weight_decay = beta1, beta2, eps, weight_decay
        self.state_bits = state_bits
        self.step = 0
        self.state: dict = {}

    @torch.no_grad()
    def update(self, model, lr: float) -> None:
        self.step += 1
        if self.state_bits == 8:
            return self._update8(model, lr)
        ps, gs, ms, vs, decays = [], [], [], [], []
        for name, p in model.named_params():
            if not p.requires_grad:
                continue
            g = p.grad
            if g is None:
                g = torch.zeros_like(p)
            elif not g.is_contiguous():
                g = g.contiguous()
            s = self.state.get(name)
            if s is None:
                s = self.state[name] = (torch.zeros_like(p), torch.zeros_like(p))
            elif isinstance(s, State8):
                s = self.state[name] = s.moments()
            ps.append(p)
            gs.append(g)
            ms.append(s[0])
            vs.append(s[1])
            decays.append(0.0 if "norm" in name else self.weight_decay)
        P.adamw_update_multi(ps, gs, ms, vs, self.step, lr, self.beta1, self.beta2, self.eps, decays)

    def _update8(self, model, lr):
        tensors = []
        for name, p in model.named_params():
            if not p.requires_grad:
                continue
            s = self.state.get(name)
            if p.numel() >= SMALL and not isinstance(s, State8):
                s = self.state[name] = State8(p) if s is None else State8.pack(*s)
            elif s is None:
                s = self.state[name] = (torch.zeros_like(p), torch.zeros_like(p))
            held = dict(state8=s.buf) if isinstance(s, State8) else dict(m=s[0], v=s[1])
            g = torch.zeros_like(p) if p.grad is None else p.grad.contiguous()
            tensors.append(dict(p=p, g=g, weight_decay=0.0 if "norm" in name else self.weight_decay, **held))
        P.adamw8_update_multi(tensors, self.step, lr, self.beta1, self.beta2, self.eps)
