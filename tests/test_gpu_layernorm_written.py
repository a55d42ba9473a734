"""GPU tests that layer norm writes every value, and none that is not finite: outputs hold
NaN before each call, every input stands between NaN, and a comparison with NaN fails.
The formulas in 64 bits and the tolerances are those of test_gpu_layernorm."""
import math

import pytest
import torch

from cpuforge_amd import ops as P
from tests.test_gpu_layernorm import BF16, DEV, DIMS, F32, U, exact, half_step, inputs

pytestmark = pytest.mark.gpu
MANY = [(4099, 576, F32), (5000, 2048, BF16), (1023, 4096, F32), (2050, 8192, BF16), (515, 16384, F32),
        (70, 40000, BF16), (20000, 17, F32), (4097, 1500, F32), (4099, 3001, BF16), (4096, 8001, BF16),
        (4101, 6000, F32), (4097, 16383, BF16), (4098, 4096, F32)]


def between_nan(t, dtype, offset=8):
    flat = torch.full((t.numel() + 2 * offset + 16,), math.nan, dtype=dtype, device=DEV)
    flat[offset:offset + t.numel()] = t.reshape(-1)
    return flat[offset:offset + t.numel()].view(t.shape)


def unwritten(*shape, dtype=F32):
    return torch.full(shape, math.nan, dtype=dtype, device=DEV)


def near(got, want, tol, what):
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (what, int((~(off <= tol)).sum()), torch.nonzero(~(off <= tol))[:5].tolist())


def run(x, w, b, dy, eps):
    rows, dim = x.shape
    y, mean, rstd = unwritten(rows, dim, dtype=x.dtype), unwritten(rows), unwritten(rows)
    P.layernorm_forward(x, w, b, y, mean, rstd, rows, dim, eps)
    dx, dw, db = unwritten(rows, dim, dtype=x.dtype), unwritten(dim), unwritten(dim)
    P.layernorm_backward(dy, x, w, mean, rstd, dx, dw, db, rows, dim, acc=False)
    return dict(y=y, mean=mean, rstd=rstd, dx=dx, dw=dw, db=db)


def check(got, x, w, b, dy, eps):
    want, tol = exact(x, w, b, dy, eps)
    near(got["y"], want["y"], tol["y"] + half_step(want["y"], x.dtype), "y")
    size = x.double().abs().mean(1)
    near(got["mean"], want["mean"], 64 * U * size, "mean")
    rstd_off = want["rstd"] * 64 * U * (1 + want["rstd"] * size)
    near(got["rstd"], want["rstd"], rstd_off, "rstd")
    # (The backward took the forward's mean and rstd, whose errors are in its tolerance as h's.)
    rel = (rstd_off / want["rstd"])[:, None]
    near(got["dx"], want["dx"], tol["dx"] + rel * want["dx"].abs() + half_step(want["dx"], x.dtype), "dx")
    near(got["dw"], want["dw"], tol["dw"] + half_step(want["dw"], F32), "dw")
    near(got["db"], want["db"], tol["db"] + half_step(want["db"], F32), "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 11])
def test_widths(rows, dim, dtype):
    eps = 1e-3 if dim < 8 else 1e-5
    x, w, b, dy = inputs(rows, dim, dtype, dim + rows)
    x, dy = between_nan(x, dtype, 8 + dim % 3), between_nan(dy, dtype, 8 + dim % 3)
    w, b = between_nan(w, F32), between_nan(b, F32)
    check(run(x, w, b, dy, eps), x, w, b, dy, eps)


@pytest.mark.parametrize("rows,dim,dtype", MANY)
def test_many_rows(rows, dim, dtype):
    x, w, b, dy = inputs(rows, dim, dtype, 3)
    x, dy = between_nan(x, dtype), between_nan(dy, dtype)
    w, b = between_nan(w, F32), between_nan(b, F32)
    check(run(x, w, b, dy, 1e-5), x, w, b, dy, 1e-5)


@pytest.mark.parametrize("rows,dim,dtype", MANY + [(11, dim, dtype) for dim in (3, 257, 769, 1025, 4097, 8193, 16385)
                                                   for dtype in (F32, BF16)])
def test_rows_beside_rows_that_are_not_finite(rows, dim, dtype):
    """Every third row NaN or infinite in x or dy: each other row has the bits that it has
    beside finite ones."""
    x, w, b, dy = inputs(rows, dim, dtype, 5)
    clean = run(x, w, b, dy, 1e-3)
    bad = torch.arange(rows, device=DEV) % 3 == 1
    x, dy = x.clone(), dy.clone()
    x[1::9], x[4::9, dim // 2], dy[7::9] = math.nan, math.inf, math.nan
    got = run(x, w, b, dy, 1e-3)
    for name in ("y", "mean", "rstd", "dx"):
        assert torch.equal(got[name][~bad], clean[name][~bad]), name
        assert bool(torch.isfinite(got[name][~bad]).all()), name
    assert bool(torch.isnan(got["y"][1::9]).all()) and bool(torch.isnan(got["dx"][bad]).all())
