"""Device-tensor entry points of the layer ops (include/cfops.h).

Each function keeps the reference op's argument meaning and its overwrite /
accumulate (+=) contract, on contiguous float32 device tensors; torch is only
the holder of device memory and the current HIP stream:

    matmul_nn / matmul_nt / matmul_tn   crates/core/src/matmul.rs:127-147
    rmsnorm_forward / rmsnorm_backward  crates/core/src/ops/rmsnorm.rs
    silu_mul_forward / silu_mul_backward crates/core/src/ops/swiglu.rs
    cross_entropy_fwd_bwd               crates/core/src/ops/loss.rs:9-55
    lm_head_ce                          crates/model/src/model.rs:436-457
      (lm_head_ce_dev: the same, its loss left in device memory)
    linear_forward / linear_backward    crates/model/src/linear.rs:56-91
      (linears_forward / linears_backward: several linears of one input)
    adamw_update                        crates/train/src/optim.rs:9-30
      (adamw_update_multi: many tensors, optim.rs:48-61)

Layers of other decoders have no reference counterpart:

    layernorm_forward / layernorm_backward
    rotary                              q and k at given positions, either layout

nor has training on preferences, rewards and a teacher:

    lm_head_logprobs(_backward)         the targets' log-probabilities
    lm_head_distill(_backward)          a loss against a teacher's top logits
    preference_loss, policy_loss        losses over them, with their gradients
    adamw8_update_multi                 AdamW with its moments in 8 bits

Misuse the reference would panic on raises `ShapeError` (an AssertionError);
library failures raise `CfattnError`.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import _lib
from .attention import Context, default_context

IGNORE_INDEX = _lib.IGNORE_INDEX


def _stream() -> int:
    """torch.cuda.current_stream().cuda_stream without the Stream object, which
    takes 5 us a call to make, half of what a small op's whole call takes."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _f32(t: torch.Tensor, name: str, numel: int | None = None) -> int:
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.float32 and t.is_contiguous() \
            and (numel is None or t.numel() == numel):
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    raise _lib.ShapeError(_lib.ERR_SHAPE,
                          f"assertion `left == right` failed: {name}.len() = {t.numel()}, expected {numel}")


_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _on(t: torch.Tensor, name: str, ctx: Context, dtypes=(torch.float32,), numel: int | None = None) -> int:
    """The address of a contiguous tensor of one of `dtypes` on the context's
    device."""
    # (A host tensor's device is -1.)
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.get_device() == ctx.device and t.is_contiguous() \
            and (numel is None or t.numel() == numel):
        return t.data_ptr()
    _check_on(t, name, ctx, dtypes)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    raise _lib.ShapeError(_lib.ERR_SHAPE,
                          f"assertion `left == right` failed: {name}.len() = {t.numel()}, expected {numel}")


def _check_on(t, name, ctx, dtypes) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name} is on device {t.get_device()}, the context on device {ctx.device}")


def _stream_of(ctx: Context) -> int:
    """The current stream of the context's device, whichever device is current."""
    return torch._C._cuda_getCurrentRawStream(ctx.device)


def _opt(t, name, numel=None):
    return None if t is None else _f32(t, name, numel)


def _targets(t: torch.Tensor, rows: int) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int64 or not t.is_contiguous():
        raise TypeError("targets must be a contiguous int64 device tensor")
    if t.numel() != rows:
        raise _lib.ShapeError(_lib.ERR_SHAPE, f"assertion `left == right` failed: targets.len() = {t.numel()}, "
                                              f"expected {rows}")
    return t.data_ptr()


def _call(ctx: Context, name: str, *args) -> None:
    _lib.check(getattr(ctx._lib, name)(ctx.handle, *args), ctx.handle)


# --------------------------------------------------------------- matmul
def _matmul(kind, a, b, c, m, k, n, acc, ctx):
    ctx = ctx or default_context()
    ka, kb = (m * k, k * n) if kind == _lib.NN else (m * k, n * k) if kind == _lib.NT else (k * m, k * n)
    _call(ctx, "cfops_matmul", kind, _f32(a, "a", ka), _f32(b, "b", kb), _f32(c, "c", m * n), m, k, n, int(acc),
          _stream())
    return c


def matmul_nn(a, b, c, m, k, n, acc=False, ctx: Context | None = None):
    """C[m,n] (+)= A[m,k] . B[k,n]"""
    return _matmul(_lib.NN, a, b, c, m, k, n, acc, ctx)


def matmul_nt(a, b, c, m, k, n, acc=False, ctx: Context | None = None):
    """C[m,n] (+)= A[m,k] . B[n,k]^T"""
    return _matmul(_lib.NT, a, b, c, m, k, n, acc, ctx)


def matmul_tn(a, b, c, m, k, n, acc=False, ctx: Context | None = None):
    """C[m,n] (+)= A[k,m]^T . B[k,n]"""
    return _matmul(_lib.TN, a, b, c, m, k, n, acc, ctx)


# -------------------------------------------------------------- RMSNorm
def rmsnorm_forward(x, w, y, rstd, rows, dim, eps, ctx: Context | None = None):
    """rmsnorm.rs:4-28: overwrites y [rows, dim] and rstd [rows]."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_rmsnorm_forward", _f32(x, "x", rows * dim), _f32(w, "w", dim), _f32(y, "y", rows * dim),
          _f32(rstd, "rstd", rows), rows, dim, float(eps), _stream())


def rmsnorm_backward(dy, x, w, rstd, dx, dw, rows, dim, ctx: Context | None = None, acc: bool = True):
    """rmsnorm.rs:33-67: accumulates into dx and dw (dw None: frozen gain), or
    overwrites them with acc=False."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_rmsnorm_grad", _f32(dy, "dy", rows * dim), _f32(x, "x", rows * dim), _f32(w, "w", dim),
          _f32(rstd, "rstd", rows), _f32(dx, "dx", rows * dim), _opt(dw, "dw", dim), rows, dim, int(acc), _stream())


# ------------------------------------------------------------ layer norm
def layernorm_forward(x, w, b, y, mean, rstd, rows, dim, eps, ctx: Context | None = None):
    """y = (x - mean) rstd w + b per row of `dim` (b None: no bias), mean and
    rstd = 1 / sqrt(var + eps): overwrites y [rows, dim], mean and rstd [rows].
    x and y are float32 or bfloat16, the others float32.  What is
    written shares memory with no other tensor."""
    ctx = ctx or default_context()
    n = rows * dim
    _call(ctx, "cfops_layernorm_forward", _code(x), _on(x, "x", ctx, _CODES, n), _on(w, "w", ctx, numel=dim),
          None if b is None else _on(b, "b", ctx, numel=dim), _on(y, "y", ctx, (x.dtype,), n),
          _on(mean, "mean", ctx, numel=rows), _on(rstd, "rstd", ctx, numel=rows), rows, dim, float(eps),
          _stream_of(ctx))


def layernorm_backward(dy, x, w, mean, rstd, dx, dw, db, rows, dim, ctx: Context | None = None, acc: bool = True):
    """Accumulates into dx (of x's type, as dy), dw and db (None: frozen), or
    overwrites them with acc=False.  They share memory with no other tensor."""
    ctx = ctx or default_context()
    n = rows * dim
    _call(ctx, "cfops_layernorm_backward", _code(x), _on(dy, "dy", ctx, (x.dtype,), n), _on(x, "x", ctx, _CODES, n),
          _on(w, "w", ctx, numel=dim), _on(mean, "mean", ctx, numel=rows), _on(rstd, "rstd", ctx, numel=rows),
          _on(dx, "dx", ctx, (x.dtype,), n), None if dw is None else _on(dw, "dw", ctx, numel=dim),
          None if db is None else _on(db, "db", ctx, numel=dim), rows, dim, int(acc), _stream_of(ctx))


def _code(t) -> int:
    """(A type that the argument checks refuse gets any.)"""
    return _CODES.get(getattr(t, "dtype", None), _lib.F32)


# ------------------------------------------------------ rotary positions
def rotary(xs, ys, cos, sin, positions=None, *, pos0: int = 0, interleaved: bool = False, inverse: bool = False,
           ctx: Context | None = None):
    """Turns tensors xs of heads [B, S, H, D] (one, or up to 4 of the same B, S and
    D, as q and k) into ys (the same shapes; a y may be its x, else it shares no
    memory with any tensor): pair i of a head's first 2 * cos.shape[1] values by cos[p, i] and
    sin[p, i] of the token's position p, (a, b) -> (a c - b s, b c + a s) (inverse:
    s negated, the gradient's way); the values behind them are copied.  The pairs
    are (i, i + half), as in the fused prologue, or (2 i, 2 i + 1) with
    `interleaved`.  positions [B, S] (int64) or pos0, pos0 + 1, ..; a position
    that the tables [max_pos, half] do not hold turns the values to NaN.  xs and ys
    are float32 or bfloat16 with any strides whose last one is 1."""
    ctx = ctx or default_context()
    if isinstance(xs, torch.Tensor):
        xs, ys = (xs,), (ys,)
    n = len(xs)
    if n != len(ys) or not 1 <= n <= _lib.ROTARY_MAX:
        raise ValueError(f"{n} xs and {len(ys)} ys: as many of either, and 1 to {_lib.ROTARY_MAX}")
    dev, table = ctx.device, b""
    x_type, y_type = getattr(xs[0], "dtype", None), getattr(ys[0], "dtype", None)
    typed, batch = x_type in _CODES and y_type in _CODES, -1
    for x, y in zip(xs, ys):
        if not (typed and isinstance(x, torch.Tensor) and isinstance(y, torch.Tensor) and x.dtype is x_type
                and y.dtype is y_type and x.get_device() == dev and y.get_device() == dev):
            _check_on(xs[0], "x", ctx, _CODES)
            _check_on(ys[0], "y", ctx, _CODES)
            _check_on(x, "x", ctx, (x_type,))
            _check_on(y, "y", ctx, (y_type,))
        shape = x.shape
        fits = y.shape == shape and len(shape) == 4
        if fits:
            b, l, heads, w = shape
            if batch < 0:
                batch, seq, dim = b, l, w
            fits = b == batch and l == seq and w == dim
        if not fits:
            raise _lib.ShapeError(_lib.ERR_SHAPE, f"x and y have shapes {tuple(shape)} and {tuple(y.shape)} beside "
                                                  f"{tuple(xs[0].shape)} ([B, S, H, D], the same but for H)")
        x0, x1, x2, x3 = x.stride()
        y0, y1, y2, y3 = y.stride()
        if (x3 != 1 or y3 != 1) and dim > 1:
            raise ValueError("the last stride of x and y must be 1")
        if not (y0 and y1 and y2) and ((y0 == 0 and b > 1) or (y1 == 0 and l > 1) or (y2 == 0 and heads > 1)):
            raise ValueError("y must not be expanded")
        table += _ROTARY_TENSOR(x.data_ptr(), y.data_ptr(), heads, x0, x1, x2, y0, y1, y2)
    pc, ps = _on(cos, "cos", ctx), _on(sin, "sin", ctx)
    held = cos.shape
    if len(held) != 2 or sin.shape != held:
        raise _lib.ShapeError(_lib.ERR_SHAPE, f"cos and sin have shapes {tuple(cos.shape)} and {tuple(sin.shape)}, "
                                              "expected [max_pos, half]")
    at = None if positions is None else _on(positions, "positions", ctx, (torch.int64,), batch * seq)
    if pos0 < 0:
        raise ValueError("pos0 must not be negative")
    max_pos, half = held
    _call(ctx, "cfops_rotary", table, n, _CODES[x_type], _CODES[y_type], batch, seq, dim, half, pc, ps,
          max_pos, at, pos0, interleaved, inverse, _stream_of(ctx))


_ROTARY_TENSOR = struct.Struct("@PPN6q").pack  # cfops_rotary_tensor


# --------------------------------------------------------------- SwiGLU
def silu_mul_forward(g, u, h, ctx: Context | None = None):
    """swiglu.rs:10-16: h = silu(g) * u (overwritten)."""
    ctx = ctx or default_context()
    n = g.numel()
    _call(ctx, "cfops_silu_mul_forward", _f32(g, "g"), _f32(u, "u", n), _f32(h, "h", n), n, _stream())


def silu_mul_backward(dh, g, u, dg, du, ctx: Context | None = None, acc: bool = True):
    """swiglu.rs:18-30: accumulates into dg and du, or overwrites them with acc=False."""
    ctx = ctx or default_context()
    n = g.numel()
    _call(ctx, "cfops_silu_mul_grad", _f32(dh, "dh", n), _f32(g, "g"), _f32(u, "u", n), _f32(dg, "dg", n),
          _f32(du, "du", n), n, int(acc), _stream())


# -------------------------------------------------------- cross-entropy
def cross_entropy_fwd_bwd(logits, targets, dlogits, rows, vocab, ctx: Context | None = None) -> float:
    """loss.rs:9-55: returns the mean loss; dlogits overwritten (may be
    logits itself).  Waits for the stream, as the reference returns the
    loss.  A target out of range raises CfattnError (the reference panics)."""
    ctx = ctx or default_context()
    loss = C.c_float(0.0)
    _call(ctx, "cfops_cross_entropy_fwd_bwd", _f32(logits, "logits", rows * vocab), _targets(targets, rows),
          _f32(dlogits, "dlogits", rows * vocab), rows, vocab, C.byref(loss), _stream())
    return loss.value


def lm_head_ce(hn, head, targets, t, d, vocab, dhn, dhead=None, ctx: Context | None = None) -> float:
    """The LM head and loss of Model::forward_backward (model.rs:436-457):
    logits = hn . head^T, mean cross-entropy, dhn = dlogits . head
    (overwritten) and dhead += dlogits^T . hn when dhead is given.  Returns
    the loss; the [t, vocab] logits are formed a chunk of rows at a time."""
    ctx = ctx or default_context()
    loss = C.c_float(0.0)
    _call(ctx, "cfops_lm_head_ce", _f32(hn, "hn", t * d), _f32(head, "head", vocab * d), _targets(targets, t), t, d,
          vocab, _f32(dhn, "dhn", t * d), _opt(dhead, "dhead", vocab * d), C.byref(loss), _stream())
    return loss.value


CE_RESULT_WORDS = 3  # cfops_ce_result: n_valid, bad_row (int32), loss (float32)
_NO_BAD_ROW = 2 ** 31 - 1


def ce_result_buffer(device) -> torch.Tensor:
    """A device block for lm_head_ce_dev's result (cfops_ce_result)."""
    return torch.empty(CE_RESULT_WORDS, dtype=torch.int32, device=device)


def ce_result_loss(result: torch.Tensor) -> torch.Tensor:
    """The loss of a cfops_ce_result block, as a 0-d float32 device tensor
    (a view of the block)."""
    return result.view(torch.float32)[2]


def lm_head_ce_dev(hn, head, targets, t, d, vocab, dhn, dhead, result, ctx: Context | None = None) -> None:
    """lm_head_ce queued on the current stream with no host wait: the loss
    block goes to `result` (ce_result_buffer), for a step captured in a HIP
    graph.  The target check is the caller's, after the stream drains
    (ce_check)."""
    ctx = ctx or default_context()
    if not isinstance(result, torch.Tensor) or not result.is_cuda or result.dtype != torch.int32 \
            or result.numel() < CE_RESULT_WORDS or not result.is_contiguous():
        raise TypeError("result must be a contiguous int32 device tensor of 3 words")
    _call(ctx, "cfops_lm_head_ce_dev", _f32(hn, "hn", t * d), _f32(head, "head", vocab * d), _targets(targets, t), t,
          d, vocab, _f32(dhn, "dhn", t * d), _opt(dhead, "dhead", vocab * d), result.data_ptr(), _stream())


def ce_check(result: torch.Tensor, targets: torch.Tensor, vocab: int) -> None:
    """Waits for `result` (a cfops_ce_result written by lm_head_ce_dev) and
    raises, with lm_head_ce's error, for a target outside [0, vocab)."""
    bad = int(result[1].item())
    if bad != _NO_BAD_ROW:
        t = int(targets.reshape(-1)[bad].item())
        raise _lib.CfattnError(_lib.ERR_ARG, f"target {t} out of range for vocab {vocab}")


def set_head_chunk_limit(nbytes: int, ctx: Context | None = None) -> None:
    ctx = ctx or default_context()
    _call(ctx, "cfops_set_head_chunk_limit", int(nbytes))


# --------------------------------------------------------------- Linear
def linear_forward(x, w, t, inn, out, y, lora_a=None, lora_b=None, lora_scale=1.0, xs=None, ctx: Context | None = None):
    """Linear::forward (linear.rs:56-71): y = x W^T (+ xs B^T with xs =
    scale * x A^T when an adapter is given); y and xs overwritten."""
    ctx = ctx or default_context()
    r = 0 if lora_a is None else lora_a.shape[0]
    _call(ctx, "cfops_linear_forward", _f32(x, "x", t * inn), _f32(w, "w", out * inn), _opt(lora_a, "lora_a", r * inn),
          _opt(lora_b, "lora_b", out * r), float(lora_scale), t, inn, out, r, _f32(y, "y", t * out),
          _opt(xs, "xs", t * r), _stream())


def linear_backward(x, xs, dy, w, t, inn, out, dx, gw=None, ga=None, gb=None, lora_a=None, lora_b=None,
                    lora_scale=1.0, ctx: Context | None = None):
    """Linear::backward (linear.rs:73-91): accumulates into dx and every
    gradient given (None: frozen)."""
    ctx = ctx or default_context()
    r = 0 if lora_a is None else lora_a.shape[0]
    _call(ctx, "cfops_linear_backward", _f32(x, "x", t * inn), _opt(xs, "xs", t * r), _f32(dy, "dy", t * out),
          _f32(w, "w", out * inn), _opt(lora_a, "lora_a", r * inn), _opt(lora_b, "lora_b", out * r),
          float(lora_scale), t, inn, out, r, _f32(dx, "dx", t * inn), _opt(gw, "gw", out * inn),
          _opt(ga, "ga", r * inn), _opt(gb, "gb", out * r), _stream())


def _linears(lins, t, inn, forward):
    """The cfops_linear array of `lins` (dicts; see linears_forward / _backward)."""
    arr = (_lib.LinearC * len(lins))()
    for c, li in zip(arr, lins):
        w, a, b = li["w"], li.get("lora_a"), li.get("lora_b")
        out = w.shape[0]
        r = 0 if a is None else a.shape[0]
        c.w, c.out, c.rank, c.lora_scale = _f32(w, "w", out * inn), out, r, float(li.get("scale", 1.0))
        c.lora_a, c.lora_b = _opt(a, "lora_a", r * inn), _opt(b, "lora_b", out * r)
        c.xs = _opt(li.get("xs"), "xs", t * r)
        if forward:
            c.y = _f32(li["y"], "y", t * out)
        else:
            c.dy = _f32(li["dy"], "dy", t * out)
            c.gw = _opt(li.get("gw"), "gw", out * inn)
            c.ga, c.gb = _opt(li.get("ga"), "ga", r * inn), _opt(li.get("gb"), "gb", out * r)
    return arr


def linears_forward(x, t, inn, lins, ctx: Context | None = None):
    """linear_forward of several linears of one input x [t, inn] in the
    launches of one.  Each is a dict of w [out, inn], y [t, out] (overwritten)
    and, with an adapter, lora_a, lora_b, scale and xs [t, rank] (overwritten)."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_linears_forward", _f32(x, "x", t * inn), t, inn, _linears(lins, t, inn, True), len(lins),
          _stream())


def linears_backward(x, t, inn, dx, lins, acc=True, ctx: Context | None = None):
    """linear_backward of several linears of one input: dicts of w, dy, gw and,
    with an adapter, lora_a, lora_b, scale, xs, ga and gb (None or absent:
    frozen; dx None: x needs no gradient).  Adds to dx and the gradients, or
    overwrites them with acc=False."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_linears_backward", _f32(x, "x", t * inn), t, inn, _opt(dx, "dx", t * inn),
          _linears(lins, t, inn, False), len(lins), int(acc), _stream())


# ---------------------------------------------------------------- AdamW
def adamw_update(p, g, m, v, t, lr, beta1, beta2, eps, weight_decay, ctx: Context | None = None):
    """optim.rs:9-30: one AdamW step (t 1-based), in place on p, m, v."""
    ctx = ctx or default_context()
    n = p.numel()
    _call(ctx, "cfops_adamw_update", _f32(p, "p"), _f32(g, "g", n), _f32(m, "m", n), _f32(v, "v", n), n, int(t),
          float(lr), float(beta1), float(beta2), float(eps), float(weight_decay), _stream())


def adamw_update_multi(ps, gs, ms, vs, t, lr, beta1, beta2, eps, weight_decays, ctx: Context | None = None):
    """adamw_update of many tensors, each with its own weight decay, in few
    launches (tensors that share memory are updated in order)."""
    ctx = ctx or default_context()
    k = len(ps)
    for name, xs in (("g", gs), ("m", ms), ("v", vs), ("weight_decays", weight_decays)):
        if len(xs) != k:
            raise _lib.ShapeError(_lib.ERR_SHAPE, f"assertion `left == right` failed: {len(xs)} {name} for {k} tensors")
    sizes = [x.numel() for x in ps]
    arrs = []
    for name, ts in (("p", ps), ("g", gs), ("m", ms), ("v", vs)):
        for x, n in zip(ts, sizes):
            # _f32's checks, spelled out once for the common case.
            if not (x.is_cuda and x.dtype is torch.float32 and x.is_contiguous() and x.numel() == n):
                _f32(x, name, n)
        arrs.append((C.c_void_p * k)(*[x.data_ptr() for x in ts]))
    _call(ctx, "cfops_adamw_update_multi", k, *arrs, (C.c_size_t * k)(*sizes), (C.c_float * k)(*weight_decays),
          int(t), float(lr), float(beta1), float(beta2), float(eps), _stream())


# ---------------------------------- log-probabilities through the LM head
def _result(t: torch.Tensor, words: int) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or t.numel() < words \
            or not t.is_contiguous():
        raise TypeError(f"result must be a contiguous int32 device tensor of {words} words")
    return t.data_ptr()


def lm_head_logprobs(hn, head, targets, t, d, vocab, logp, lse, result, keep=None, ctx: Context | None = None) -> None:
    """logits = hn . head^T (never held whole); lse [t] is their log-sum-exp and
    logp [t] the targets' logits less it, both 0 where the target is
    IGNORE_INDEX (all overwritten).  `result` (ce_result_buffer) gets the mean
    of -logp (ce_result_loss) and the first row whose target is out of range,
    which ce_check reports; such a row's logp is NaN.  `keep` (a uint8 tensor of
    lm_head_logprobs_keep_bytes, when given) takes what the backward reads.  No
    host wait."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_lm_head_logprobs", _f32(hn, "hn", t * d), _f32(head, "head", vocab * d), _targets(targets, t),
          t, d, vocab, _f32(logp, "logp", t), _f32(lse, "lse", t), _result(result, CE_RESULT_WORDS), *_keep(keep),
          _stream())


def lm_head_logprobs_backward(hn, head, targets, lse, dlogp, t, d, vocab, dhn=None, dhead=None, keep=None,
                              ctx: Context | None = None, acc: bool = True) -> None:
    """From the gradient dlogp of logp: dhn (overwritten) and dhead +=
    dlogits^T . hn (acc=False: overwritten), each when given.  hn, head, targets, lse and keep are the
    forward's; without keep the logits are formed again."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_lm_head_logprobs_backward", _f32(hn, "hn", t * d), _f32(head, "head", vocab * d),
          _targets(targets, t), _f32(lse, "lse", t), _f32(dlogp, "dlogp", t), t, d, vocab, _opt(dhn, "dhn", t * d),
          _opt(dhead, "dhead", vocab * d), int(acc), *_keep(keep), _stream())


def _keep(keep):
    if keep is None:
        return None, 0
    if not isinstance(keep, torch.Tensor) or not keep.is_cuda or keep.dtype != torch.uint8 or not keep.is_contiguous():
        raise TypeError("keep must be a contiguous uint8 device tensor")
    return keep.data_ptr(), keep.numel()


def lm_head_logprobs_keep_bytes(t: int, d: int, vocab: int) -> int:
    """Size of lm_head_logprobs' keep (about 4 t vocab + 4 d vocab bytes), 0
    where it uses none."""
    return _lib.lib().cfops_lm_head_logprobs_keep_bytes(int(t), int(d), int(vocab))


# ------------------------------ distillation from a teacher's top logits
def lm_head_distill(hn, head, ids, teacher, t, d, vocab, k, loss, result, teacher_lse=None, temperature=1.0, keep=None,
                    ctx: Context | None = None) -> None:
    """The loss [t] (overwritten) of the student's logits x = hn . head^T /
    temperature (never held whole), q = softmax(x), against a teacher's top
    logits: of each row k tokens ids [t, k] (int64) and their logits teacher [t, k];
    those with id IGNORE_INDEX or logit -inf are not there.  With p =
    exp(teacher / temperature - L)
        sum p (log p - log q) + p_rest (log p_rest - log q_rest),
    L = teacher_lse [t], the log-sum-exp of all the teacher's logits / temperature,
    and the other tokens (the rest) one class; teacher_lse None: L the entries' own,
    and no rest.  A row without entries has loss 0.  `result` (ce_result_buffer) gets
    the mean (ce_result_loss) and the first row with a token out of range or
    twice, or a teacher's value NaN or +inf, which distill_check reports; such a
    row's loss is NaN.  `keep` (a uint8 tensor of lm_head_distill_keep_bytes, when
    given) takes what the backward reads.  No host wait."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_lm_head_distill", *_distill(hn, head, ids, teacher, teacher_lse, t, d, vocab, k, ctx), t, d,
          vocab, k, float(temperature), _on(loss, "loss", ctx, numel=t), _result(_here(result, ctx), CE_RESULT_WORDS),
          *_keep(_here(keep, ctx)), _stream_of(ctx))


def lm_head_distill_backward(hn, head, ids, teacher, dloss, t, d, vocab, k, dhn=None, dhead=None, teacher_lse=None,
                             temperature=1.0, keep=None, ctx: Context | None = None, acc: bool = True) -> None:
    """From the gradient dloss of loss: dhn (overwritten) and dhead += (acc=False:
    overwritten), each when given.  The others are the forward's; without keep the
    logits are formed again."""
    ctx = ctx or default_context()
    _call(ctx, "cfops_lm_head_distill_backward", *_distill(hn, head, ids, teacher, teacher_lse, t, d, vocab, k, ctx),
          _on(dloss, "dloss", ctx, numel=t), t, d, vocab, k, float(temperature),
          None if dhn is None else _on(dhn, "dhn", ctx, numel=t * d),
          None if dhead is None else _on(dhead, "dhead", ctx, numel=vocab * d), int(acc), *_keep(_here(keep, ctx)),
          _stream_of(ctx))


def _here(t, ctx):
    """t, or its error where it is a tensor of another device than the context's."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() != ctx.device:
        raise ValueError(f"a buffer is on device {t.get_device()}, the context on device {ctx.device}")
    return t


def _distill(hn, head, ids, teacher, lse, t, d, vocab, k, ctx):
    return (_on(hn, "hn", ctx, numel=t * d), _on(head, "head", ctx, numel=vocab * d),
            _on(ids, "ids", ctx, (torch.int64,), t * k), _on(teacher, "teacher", ctx, numel=t * k),
            None if lse is None else _on(lse, "teacher_lse", ctx, numel=t))


def lm_head_distill_keep_bytes(t: int, d: int, vocab: int, k: int) -> int:
    """Size of lm_head_distill's keep."""
    return _lib.lib().cfops_lm_head_distill_keep_bytes(int(t), int(d), int(vocab), int(k))


def distill_check(result: torch.Tensor) -> None:
    """Waits for `result` and raises for a row whose entries lm_head_distill does
    not take."""
    bad = int(result[1].item())
    if bad != _NO_BAD_ROW:
        raise _lib.CfattnError(_lib.ERR_ARG, f"row {bad} names a token out of range or twice, or a value of the "
                                             "teacher's is NaN or +inf")


# ------------------------------------------- losses over packed sequences
PREFERENCE_FORMS = {"sigmoid": 0, "hinge": 1, "squared": 2}
POLICY_REDUCTIONS = {"token": 0, "sequence": 1}
PREFERENCE_RESULT_WORDS, POLICY_RESULT_WORDS = 4, 5


class PreferenceResult(NamedTuple):
    """Views of a cfops_preference_result block, 0-d device tensors."""
    loss: torch.Tensor
    accuracy: torch.Tensor
    margin: torch.Tensor


class PolicyResult(NamedTuple):
    """Views of a cfops_policy_result block, 0-d device tensors."""
    loss: torch.Tensor
    kl: torch.Tensor
    clipped: torch.Tensor
    n_scored: torch.Tensor


def preference_result(result: torch.Tensor) -> PreferenceResult:
    return PreferenceResult(*result.view(torch.float32)[1:4].unbind())


def policy_result(result: torch.Tensor) -> PolicyResult:
    return PolicyResult(*result.view(torch.float32)[2:5].unbind(), result[0])


def _bad_seq(bad: int) -> None:
    if bad != _NO_BAD_ROW:
        raise _lib.CfattnError(_lib.ERR_ARG, f"offsets of sequence {bad} do not rise within the rows")


def preference_check(result: torch.Tensor) -> None:
    """Waits for `result` and raises where a sequence's offsets do not rise
    within the rows."""
    _bad_seq(int(result[0].item()))


def policy_check(result: torch.Tensor) -> None:
    _bad_seq(int(result[1].item()))


def _offsets(t: torch.Tensor) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int64 or not t.is_contiguous():
        raise TypeError("offsets must be a contiguous int64 device tensor")
    return t.data_ptr()


def preference_loss(logp, ref_logp, targets, offsets, dlogp, rewards, result, *, beta: float, form: str = "sigmoid",
                    margin: float = 0.0, label_smoothing: float = 0.0, length_mean: bool = False,
                    ctx: Context | None = None) -> None:
    """The mean loss of pairs of sequences and its gradient dlogp.  Sequence i
    is rows [offsets[i], offsets[i + 1]) of logp; 2j is the chosen and 2j + 1
    the rejected one of pair j.  A reward is beta times the sum (length_mean:
    the mean) of logp - ref_logp over a sequence's scored rows, those whose
    target is not IGNORE_INDEX (targets None: all; ref_logp None: of logp).
    With z = chosen - rejected reward - margin:
        "sigmoid"  -(1 - s) log sigmoid(z) - s log sigmoid(-z), s = label_smoothing
        "hinge"    max(0, 1 - z)
        "squared"  (z - 1/2)^2
    rewards [2 * pairs] and `result` (at least PREFERENCE_RESULT_WORDS int32; see
    preference_result, preference_check) are overwritten, and dlogp in the rows
    of sequences.  No host wait."""
    ctx = ctx or default_context()
    rows, entries = logp.numel(), offsets.numel()
    if entries % 2 == 0:
        raise _lib.ShapeError(_lib.ERR_SHAPE, f"offsets of pairs have an odd number of entries, got {entries}")
    if form not in PREFERENCE_FORMS:
        raise ValueError(f"unknown preference form {form!r}")
    tp = None if targets is None else _targets(targets, rows)
    _call(ctx, "cfops_preference_loss", _f32(logp, "logp"), _opt(ref_logp, "ref_logp", rows), tp, rows,
          _offsets(offsets), entries // 2, PREFERENCE_FORMS[form], float(beta), float(margin), float(label_smoothing),
          int(length_mean), _f32(dlogp, "dlogp", rows), _f32(rewards, "rewards", entries - 1),
          _result(result, PREFERENCE_RESULT_WORDS), _stream())


def policy_loss(logp, old_logp, ref_logp, advantages, targets, offsets, dlogp, result, *, clip_low: float,
                clip_high: float, kl_coef: float = 0.0, reduction: str = "token", per_token: bool | None = None,
                ctx: Context | None = None) -> None:
    """The clipped policy loss of sequences (as in preference_loss) and its
    gradient dlogp: with r = exp(logp - old_logp) (None: r = 1) and the
    advantage A of its sequence (advantages [sequences]) or of the row ([rows];
    per_token says which where the two numbers are the same), a scored row's
    loss is
        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef k,
        k = exp(ref_logp - logp) - (ref_logp - logp) - 1  (ref_logp None: none),
    averaged over the scored rows ("token") or over the sequences' means
    ("sequence").  `result` (at least POLICY_RESULT_WORDS int32; see
    policy_result, policy_check) is overwritten, and dlogp in the rows of
    sequences.  No host wait."""
    ctx = ctx or default_context()
    rows, seqs = logp.numel(), offsets.numel() - 1
    if seqs < 0:
        raise _lib.ShapeError(_lib.ERR_SHAPE, "offsets of sequences have one entry more than those, got none")
    if reduction not in POLICY_REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r}")
    if per_token is None:
        per_token = advantages.numel() != seqs
    tp = None if targets is None else _targets(targets, rows)
    _call(ctx, "cfops_policy_loss", _f32(logp, "logp"), _opt(old_logp, "old_logp", rows),
          _opt(ref_logp, "ref_logp", rows), _f32(advantages, "advantages", rows if per_token else seqs), tp, rows,
          _offsets(offsets), seqs, int(per_token), float(clip_low), float(clip_high), float(kl_coef),
          POLICY_REDUCTIONS[reduction], _f32(dlogp, "dlogp", rows), _result(result, POLICY_RESULT_WORDS), _stream())


# ------------------------------------------- AdamW with states in 8 bits
def adamw8_state(n: int, device="cuda") -> torch.Tensor:
    """An 8-bit state of n values (cfops_adamw_tensor), zero moments."""
    return torch.zeros(_lib.lib().cfops_adamw8_state_bytes(int(n)), dtype=torch.uint8, device=device)


def _state8(s: torch.Tensor, n: int) -> int:
    if not isinstance(s, torch.Tensor) or not s.is_cuda or s.dtype != torch.uint8 or not s.is_contiguous():
        raise TypeError("state8 must be a contiguous uint8 device tensor")
    want = _lib.lib().cfops_adamw8_state_bytes(n)
    if s.numel() != want:
        raise _lib.ShapeError(_lib.ERR_SHAPE, f"assertion `left == right` failed: state8.len() = {s.numel()}, "
                                              f"expected {want}")
    return s.data_ptr()


class Adamw8Tensors:
    """The tensors of adamw8_update_multi, checked once: a list of dicts of p,
    g, weight_decay and either m and v or state8 (adamw8_state; with m and v
    too, they are what adamw8_pack_multi reads and adamw8_unpack_multi writes).
    It keeps the tensors alive; a table may be passed any number of times."""

    def __init__(self, tensors):
        self.tensors = list(tensors)
        self.table = (_lib.AdamwTensorC * len(self.tensors))()
        for c, t in zip(self.table, self.tensors):
            p, g, m, v, s = (t.get(k) for k in ("p", "g", "m", "v", "state8"))
            if s is None and (m is None or v is None):
                raise ValueError("a tensor needs m and v, or state8")
            of = next((x for x in (p, m, v) if x is not None), None)
            if of is None:
                raise ValueError("a tensor needs p, or m and v")
            n = of.numel()
            c.p, c.g, c.m, c.v = (_opt(x, k, n) for x, k in ((p, "p"), (g, "g"), (m, "m"), (v, "v")))
            c.state8 = None if s is None else _state8(s, n)
            c.n, c.weight_decay = n, float(t.get("weight_decay", 0.0))


def _adamw8(name, tensors, ctx, *args):
    ctx = ctx or default_context()
    table = tensors if isinstance(tensors, Adamw8Tensors) else Adamw8Tensors(tensors)
    _call(ctx, name, len(table.tensors), table.table, *args, _stream())


def adamw8_update_multi(tensors, t, lr, beta1, beta2, eps, ctx: Context | None = None) -> None:
    """One AdamW step (t 1-based) of many tensors (Adamw8Tensors, or a list it
    takes), those with a state8 with their moments held in 8 bits, the others
    as adamw_update.  In place, in few launches."""
    _adamw8("cfops_adamw8_update_multi", tensors, ctx, int(t), float(lr), float(beta1), float(beta2), float(eps))


def adamw8_pack_multi(tensors, ctx: Context | None = None) -> None:
    """The f32 moments m and v of the tensors that have a state8 into it."""
    _adamw8("cfops_adamw8_pack_multi", tensors, ctx)


def adamw8_unpack_multi(tensors, ctx: Context | None = None) -> None:
    """The moments that 8-bit states stand for, into m and v."""
    _adamw8("cfops_adamw8_unpack_multi", tensors, ctx)
