"""GPU tests of layer norm, forward and backward, against the formulas in 64
bits.

Tolerances count roundings of 32 bits (u = 2^-24 each): a lane adds up at most
32 values of a row one after the other, then 6 levels of a wave and 8 of a
workgroup, so that a row's sums are off by less than 64 u of the sum of their
terms' sizes; everything after is a handful of roundings.  A bf16 result adds
half a step of its own, 2^-8 of its size."""
import pytest
import torch

from cpuforge_amd import autograd as A
from cpuforge_amd import ops as P
from cpuforge_amd._lib import CfattnError, ShapeError

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def inputs(rows, dim, dtype, seed=0, shift=0.0, offset=0):
    """`offset`: how many values x and dy start off their allocation."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def placed(t):
        flat = torch.zeros(t.numel() + offset + 9, dtype=dtype, device=DEV)
        flat[offset:offset + t.numel()] = t.reshape(-1).to(dtype)
        return flat[offset:offset + t.numel()].view(t.shape)
    x = placed(rand(rows, dim) * torch.exp(0.5 * rand(rows, 1)) + shift + 0.3 * rand(rows, 1))
    dy = placed(0.1 * rand(rows, dim))
    return x, 1 + 0.3 * rand(dim), 0.2 * rand(dim), dy


def half_step(t, dtype):
    return (2.0 ** -8 if dtype == BF16 else U) * t.abs()


def exact(x, w, b, dy, eps):
    x, w, dy = x.double(), w.double(), dy.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / (((x - mean) ** 2).mean(1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    y = h * w + (b.double() if b is not None else 0)
    g = dy * w
    m0, m1 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - m0 - h * m1)
    # How far h may be off, and with it what is formed of it.
    eh = U * (64 * rstd * x.abs().mean(1, keepdim=True) + 64 * h.abs())
    tol = dict(y=eh * w.abs() + U * (3 * y.abs() + (b.abs() if b is not None else 0)),
               dx=rstd * (64 * U * (g.abs() + g.abs().mean(1, keepdim=True)
                                    + h.abs() * (g * h).abs().mean(1, keepdim=True))
                          + eh * m1.abs() + h.abs() * (g.abs() * eh).mean(1, keepdim=True)) + 64 * U * dx.abs())
    n = 64 + x.shape[0] / 512  # rows one after the other, then the parts
    tol["dw"] = (n * U * (dy * h).abs() + dy.abs() * eh).sum(0)
    tol["db"] = (n * U * dy.abs()).sum(0)
    return dict(y=y, mean=mean[:, 0], rstd=rstd[:, 0], dx=dx, dw=(dy * h).sum(0), db=dy.sum(0)), tol


def near(got, want, tol, what):
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() - tol).max()))


def forward(x, w, b, eps):
    rows, dim = x.shape
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    P.layernorm_forward(x, w, b, y, mean, rstd, rows, dim, eps)
    return y, mean, rstd


# The widths at which a row takes another number of waves or chunks, by one more or less.
DIMS = [1, 2, 3, 5, 63, 64, 255, 256, 257, 511, 576, 769, 1001, 1024, 1025, 1536, 2048, 2049, 3001, 4096, 4097, 5000,
        8192, 8193, 12001, 16384, 16385, 33000]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 11])
def test_forward_and_backward(rows, dim, dtype):
    eps = 1e-3 if dim < 8 else 1e-5  # (of a row of few values the variance may be next to nothing)
    bias = dim % 2 == 0
    x, w, b, dy = inputs(rows, dim, dtype, dim + rows, offset=dim % 3)
    b = b if bias else None
    want, tol = exact(x, w, b, dy, eps)
    y, mean, rstd = forward(x, w, b, eps)
    near(y, want["y"], tol["y"] + half_step(want["y"], dtype), "y")
    near(mean, want["mean"], 64 * U * x.double().abs().mean(1), "mean")
    near(rstd, want["rstd"], want["rstd"] * 64 * U * (1 + want["rstd"] * x.double().abs().mean(1)), "rstd")
    # Overwriting, and adding to what is there.
    for acc in (False, True):
        g = torch.Generator(device=DEV).manual_seed(5)
        dx = torch.randn(rows, dim, generator=g, device=DEV).to(dtype)
        dw, db = torch.randn(2, dim, generator=g, device=DEV).unbind()
        was = [t.double() if acc else torch.zeros_like(t).double() for t in (dx, dw, db)]
        kept = db.clone()
        P.layernorm_backward(dy, x, w, want["mean"].float(), want["rstd"].float(), dx, dw, db if bias else None, rows,
                             dim, acc=acc)
        for name, got, w0 in zip(("dx", "dw", "db"), (dx, dw, db), was):
            if name == "db" and not bias:
                assert torch.equal(db, kept)
                continue
            sum_ = want[name] + w0
            near(got, sum_, tol[name] + half_step(sum_, dtype if name == "dx" else F32), (name, acc))


@pytest.mark.parametrize("rows,dim,dtype", [(4099, 576, F32), (5000, 2048, BF16), (1023, 4096, F32), (2050, 8192, BF16),
                                            (515, 16384, F32), (70, 40000, BF16), (20000, 17, F32),
                                            # Two rows at a time, in either number of waves.
                                            (4097, 1500, F32), (4099, 3001, BF16), (4096, 8001, BF16), (4101, 6000, F32),
                                            (4097, 16383, BF16), (4098, 4096, F32)])
def test_many_rows(rows, dim, dtype):
    x, w, b, dy = inputs(rows, dim, dtype, 3)
    want, tol = exact(x, w, b, dy, 1e-5)
    y, mean, rstd = forward(x, w, b, 1e-5)
    near(y, want["y"], tol["y"] + half_step(want["y"], dtype), "y")
    dx, dw, db = torch.empty_like(x), torch.empty(dim, device=DEV), torch.empty(dim, device=DEV)
    P.layernorm_backward(dy, x, w, mean, rstd, dx, dw, db, rows, dim, acc=False)
    near(dx, want["dx"], tol["dx"] + half_step(want["dx"], dtype), "dx")
    near(dw, want["dw"], tol["dw"] + half_step(want["dw"], F32), "dw")
    near(db, want["db"], tol["db"] + half_step(want["db"], F32), "db")
    # The same bits again.
    again = [torch.empty_like(t) for t in (dx, dw, db)]
    P.layernorm_backward(dy, x, w, mean, rstd, *again, rows, dim, acc=False)
    assert all(torch.equal(a, c) for a, c in zip(again, (dx, dw, db)))
    # A frozen weight or bias changes nothing in the others.
    P.layernorm_backward(dy, x, w, mean, rstd, again[0], None, again[2].zero_(), rows, dim, acc=False)
    assert torch.equal(again[0], dx) and torch.equal(again[2], db)
    P.layernorm_backward(dy, x, w, mean, rstd, again[0].zero_(), None, None, rows, dim, acc=False)
    assert torch.equal(again[0], dx)


def test_rows_far_from_zero():
    """The deviations are from the mean itself: 4096 + noise has all the bits that its
    values have (x is a multiple of 2^-11 there, the mean is off by up to 64 u of it)."""
    x, w, b, _ = inputs(64, 576, F32, 9, shift=4096.0)
    want, tol = exact(x, w, b, x, 1e-5)
    y, *_ = forward(x, w, b, 1e-5)
    near(y, want["y"], tol["y"], "y")


def test_rows_without_deviation_and_not_finite_ones():
    x, w, b, dy = inputs(12, 700, F32, 2)
    x[3] = 1.5
    x[5, 10] = float("inf")
    x[7, 0] = float("nan")
    x[9] = 0.0
    y, mean, rstd = forward(x, w, b, 1e-5)
    fine = [i for i in range(12) if i not in (5, 7)]
    want, tol = exact(x[fine], w, b, dy[fine], 1e-5)
    near(y[fine], want["y"], tol["y"], "y")
    assert bool((y[3] == b).all()) and bool((y[9] == b).all())
    assert bool(torch.isnan(y[5]).all()) and bool(torch.isnan(y[7]).all())
    dx = torch.empty_like(x)
    P.layernorm_backward(dy, x, w, mean, rstd, dx, None, None, 12, 700, acc=False)
    near(dx[fine], want["dx"], tol["dx"], "dx")
    assert bool(torch.isnan(dx[5]).all()) and bool(torch.isnan(dx[7]).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [7, 576, 2050, 9000, 40000])
def test_nothing_is_written_behind_the_rows(dim, dtype):
    x, w, b, dy = inputs(5, dim, dtype)
    rows = 4
    flat = [torch.full((rows * dim + 64,), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    stats = [torch.full((rows + 8,), 7.0, device=DEV) for _ in range(2)]
    sums = [torch.full((dim + 8,), 7.0, device=DEV) for _ in range(2)]
    y, dx = (f[:rows * dim].view(rows, dim) for f in flat)
    mean, rstd = (s[:rows] for s in stats)
    dw, db = (s[:dim] for s in sums)
    P.layernorm_forward(x[:rows], w, b, y, mean, rstd, rows, dim, 1e-5)
    P.layernorm_backward(dy[:rows], x[:rows], w, mean, rstd, dx, dw, db, rows, dim, acc=False)
    for f, n in zip((*flat, *stats, *sums), (rows * dim, rows * dim, rows, rows, dim, dim)):
        assert bool((f[n:] == 7.0).all())


def test_no_rows():
    w = torch.ones(30, device=DEV)
    e, s = torch.empty(0, 30, device=DEV), torch.empty(0, device=DEV)
    dw, db = torch.ones(30, device=DEV), torch.ones(30, device=DEV)
    P.layernorm_forward(e, w, w, e, s, s, 0, 30, 1e-5)
    P.layernorm_backward(e, e, w, s, s, e, dw, db, 0, 30)
    assert bool((dw == 1).all()) and bool((db == 1).all())
    P.layernorm_backward(e, e, w, s, s, e, dw, db, 0, 30, acc=False)
    assert not dw.any() and not db.any()
    x = torch.zeros(0, 30, device=DEV, requires_grad=True)
    A.layer_norm(x, w.requires_grad_(), None, 1e-5).sum().backward()
    assert x.grad.shape == (0, 30) and not w.grad.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd(dtype):
    x, w, b, dy = inputs(60, 576, dtype)
    want, tol = exact(x, w, b, dy, 1e-5)
    x3 = x.view(3, 20, 576).clone().requires_grad_()
    w, b = w.requires_grad_(), b.requires_grad_()
    y = A.layer_norm(x3, w, b, 1e-5)
    assert y.dtype == dtype and y.shape == x3.shape
    y.backward(dy.view(3, 20, 576))
    near(x3.grad.view(60, 576), want["dx"], tol["dx"] + half_step(want["dx"], dtype), "dx")
    near(w.grad, want["dw"], tol["dw"] + half_step(want["dw"], F32), "dw")
    near(b.grad, want["db"], tol["db"] + half_step(want["db"], F32), "db")
    # Transposed and expanded inputs.
    xt = x.t().contiguous().t().requires_grad_()
    yt = A.layer_norm(xt, w, None, 1e-5)
    near(yt.detach(), want["y"] - b.double().detach(), tol["y"] + half_step(want["y"] - b.double().detach(), dtype), "y")
    gx, = torch.autograd.grad(yt, xt, torch.ones((), dtype=dtype, device=DEV).expand(60, 576))
    ones, tol1 = exact(x, w.detach(), None, torch.ones_like(x), 1e-5)
    near(gx, ones["dx"], tol1["dx"] + half_step(ones["dx"], dtype), "dx of ones")


def test_gradients_against_differences():
    """Along a direction: (f(+h) - f(-h)) / 2h of the forward itself, f = sum(y dy) summed in
    64 bits.  Each y is off by its tolerance, and the third derivative's term is h^2 times a
    number of the size of f's own values (directions are of unit deviation, rows' rstd near 1)."""
    x, w, b, dy = inputs(8, 300, F32, 4)
    g = torch.Generator(device=DEV).manual_seed(8)
    _, tol = exact(x, w, b, dy, 1e-5)
    _, mean, rstd = forward(x, w, b, 1e-5)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    P.layernorm_backward(dy, x, w, mean, rstd, dx, dw, db, 8, 300, acc=False)
    h = 2.0 ** -7

    def f(x, w, b):
        return float((forward(x, w, b, 1e-5)[0].double() * dy).sum())
    for at, grad in ((0, dx), (1, dw), (2, db)):
        v = torch.randn(grad.shape, generator=g, device=DEV)
        args = [x, w, b]
        lo, hi = ([a + s * h * v if i == at else a for i, a in enumerate(args)] for s in (-1, 1))
        slope = (f(*hi) - f(*lo)) / (2 * h)
        want = float((grad.double() * v).sum())
        size = float((dy.double().abs() * (3 * rstd[:, None].double() ** 3 + 1) * w.abs()).sum())
        noise = 2 * float((tol["y"] * dy.abs()).sum()) / (2 * h) + h * h * size
        assert abs(slope - want) <= noise, (at, slope, want, noise)


def test_captured_replays_beside_eager_calls():
    """Two graphs share the context's scratch: replayed one after the other, with eager
    calls of other sizes between, each gives its eager bits."""
    cases = [(600, 576, F32), (300, 2048, BF16)]
    runs = []
    for rows, dim, dtype in cases:
        x, w, b, dy = inputs(rows, dim, dtype, rows)
        out = [torch.empty_like(x), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV), torch.empty_like(x),
               torch.empty(dim, device=DEV), torch.empty(dim, device=DEV)]

        def step(x=x, w=w, b=b, dy=dy, out=out, rows=rows, dim=dim):
            P.layernorm_forward(x, w, b, *out[:3], rows, dim, 1e-5)
            P.layernorm_backward(dy, x, w, *out[1:3], *out[3:], rows, dim, acc=False)
        step()
        torch.cuda.synchronize()
        want = [o.clone() for o in out]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((graph, out, want, step))  # (the graph reads what the step holds)
    for rep in range(3):
        for graph, out, want, _ in runs:
            for o in out:
                o.fill_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(out, want)), rep
            x, w, b, dy = inputs(40 << rep, 4096, F32, rep)
            y, mean, rstd = forward(x, w, b, 1e-5)
            P.layernorm_backward(dy, x, w, mean, rstd, torch.empty_like(x), torch.empty_like(w), torch.empty_like(w),
                                 40 << rep, 4096, acc=False)
            torch.cuda.synchronize()


def test_side_stream():
    x, w, b, _ = inputs(50, 576, F32)
    want = forward(x, w, b, 1e-5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = forward(x, w, b, 1e-5)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_refusals():
    x, w, b, dy = inputs(4, 8, F32)
    y, s = torch.empty_like(x), torch.empty(4, device=DEV)
    ok = dict(x=x, w=w, b=b, y=y, mean=s, rstd=s.clone(), rows=4, dim=8, eps=1e-5)
    P.layernorm_forward(**ok)
    for change, error in ((dict(x=x.half()), TypeError), (dict(y=y.bfloat16()), TypeError), (dict(w=w.bfloat16()), TypeError),
                          (dict(x=x.cpu()), TypeError), (dict(x=x.t()), ValueError), (dict(rows=5), ShapeError),
                          (dict(dim=4), ShapeError), (dict(b=b[:7]), ShapeError), (dict(mean=s[:3]), ShapeError),
                          (dict(w=None), TypeError)):
        with pytest.raises(error):
            P.layernorm_forward(**{**ok, **change})
    args = dict(dy=dy, x=x, w=w, mean=s, rstd=s, dx=y, dw=w.clone(), db=b.clone(), rows=4, dim=8)
    for change, error in ((dict(dy=dy.bfloat16()), TypeError), (dict(dx=y.bfloat16()), TypeError),
                          (dict(dw=w[:7]), ShapeError), (dict(dx=None), TypeError)):
        with pytest.raises(error):
            P.layernorm_backward(**{**args, **change})
    ctx = P.default_context()
    with pytest.raises(CfattnError, match="dtype"):
        P._call(ctx, "cfops_layernorm_forward", 7, x.data_ptr(), w.data_ptr(), None, y.data_ptr(), s.data_ptr(),
                s.data_ptr(), 4, 8, 1e-5, 0)
    with pytest.raises(CfattnError, match="2\\^26"):
        P._call(ctx, "cfops_layernorm_forward", 0, x.data_ptr(), w.data_ptr(), None, y.data_ptr(), s.data_ptr(),
                s.data_ptr(), 4, 1 << 26, 1e-5, 0)
    with pytest.raises(CfattnError, match="null"):
        P._call(ctx, "cfops_layernorm_forward", 0, None, w.data_ptr(), None, y.data_ptr(), s.data_ptr(), s.data_ptr(),
                4, 8, 1e-5, 0)
