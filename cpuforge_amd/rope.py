"""RoPE tables for the fused attention prologue (crates/core/src/ops/rope.rs).

`RopeCache(head_dim, max_pos, theta, scaling)` builds the reference's cos/sin
tables [max_pos, head_dim/2] (computed in f64, rounded to f32; rope.rs:46-63)
through libcfattn's host helper; the rotation itself runs on the GPU inside
the prologue kernels, or in ops.rotary.  Beside the reference's Llama3Scaling,
LinearScaling, NtkScaling and YarnScaling stretch a table over contexts longer
than a model was trained on, for either.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _lib


@dataclass(frozen=True)
class Llama3Scaling:
    """rope.rs:16-22; `apply` is Llama3Scaling::apply (rope.rs:26-38)."""
    factor: float
    low_freq_factor: float
    high_freq_factor: float
    original_max_position: float

    def c(self) -> _lib.Llama3ScalingC:
        return _lib.Llama3ScalingC(self.factor, self.low_freq_factor, self.high_freq_factor,
                                   self.original_max_position)

    def apply(self, inv_freq: float) -> float:
        sc = self.c()
        return _lib.lib().cfattn_llama3_scale(C.byref(sc), float(inv_freq))


@dataclass(frozen=True)
class LinearScaling:
    """Positions divided by `factor`."""
    factor: float

    def c(self) -> _lib.RopeScalingC:
        return _lib.RopeScalingC(kind=1, factor=self.factor)


@dataclass(frozen=True)
class NtkScaling:
    """theta * factor^(head_dim / (head_dim - 2)): the slowest pair turns `factor`
    times slower, the fastest as before."""
    factor: float

    def c(self) -> _lib.RopeScalingC:
        return _lib.RopeScalingC(kind=2, factor=self.factor)


@dataclass(frozen=True)
class YarnScaling:
    """Pairs that turn at most beta_slow times in original_max_position positions
    turn `factor` times slower, those that turn beta_fast times or more as before,
    a line over the pairs in between; cos and sin are multiplied by
    attention_factor (None: 0.1 ln(factor) + 1, of a factor of 1 or more), which the
    scores have squared."""
    factor: float
    original_max_position: float
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def c(self) -> _lib.RopeScalingC:
        if self.attention_factor is not None and not self.attention_factor > 0:
            raise ValueError("attention_factor must be positive")
        return _lib.RopeScalingC(kind=3, factor=self.factor, original_max_position=self.original_max_position,
                                 beta_fast=self.beta_fast, beta_slow=self.beta_slow,
                                 attention_factor=self.attention_factor or 0.0)


class RopeCache:
    """rope.rs:6-12 / 41-63: cos and sin as float32 arrays [max_pos, head_dim/2].
    Where a part of each head turns (ops.rotary), head_dim is that part's."""

    def __init__(self, head_dim: int, max_pos: int, theta: float,
                 scaling: Llama3Scaling | LinearScaling | NtkScaling | YarnScaling | None = None):
        if head_dim % 2 != 0:
            raise _lib.ShapeError(_lib.ERR_SHAPE, "head_dim must be even")
        self.head_dim = head_dim
        self.half = head_dim // 2
        self.max_pos = max_pos
        self.theta = theta
        self.scaling = scaling
        self.cos = np.empty((max_pos, self.half), dtype=np.float32)
        self.sin = np.empty((max_pos, self.half), dtype=np.float32)
        sc = scaling.c() if scaling is not None else None
        table = _lib.lib().cfattn_rope_table_scaled if isinstance(sc, _lib.RopeScalingC) else \
            _lib.lib().cfattn_rope_table
        rc = table(head_dim, max_pos, float(theta), C.byref(sc) if sc is not None else None, self.cos.ctypes.data,
                   self.sin.ctypes.data)
        _lib.check(rc)

    @classmethod
    def new(cls, head_dim: int, max_pos: int, theta: float) -> "RopeCache":
        return cls(head_dim, max_pos, theta)

    @classmethod
    def with_scaling(cls, head_dim: int, max_pos: int, theta: float, scaling) -> "RopeCache":
        return cls(head_dim, max_pos, theta, scaling)
