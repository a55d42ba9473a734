"""GPU tests of ops.rotary against the formula in 64 bits over the same tables.

A turned value is two products and a sum: off by at most 2 u (|a c| + |b s|)
+ u |result| (u = 2^-24), and half a step of a bf16 result, 2^-8 of its size;
copied values are exact but for that step."""
import pytest
import torch

from cpuforge_amd import RopeCache, YarnScaling
from cpuforge_amd import autograd as A
from cpuforge_amd import device as D
from cpuforge_amd import ops as P
from cpuforge_amd._lib import CfattnError, ShapeError

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def tables(max_pos, half, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    angle = torch.rand(max_pos, half, generator=g, device=DEV) * 6.3
    return (angle.cos() * scale).contiguous(), (angle.sin() * scale).contiguous()


def rand(*shape, dtype=F32, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def exact(x, cos, sin, positions, interleaved, inverse):
    """(the turned x, what it may be off but for the output's rounding)."""
    v, half = x.double(), cos.shape[1]
    c, s = cos.double()[positions][:, :, None], sin.double()[positions][:, :, None]
    s = -s if inverse else s
    y, tol = v.clone(), torch.zeros_like(v)
    at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = v[..., at[0]], v[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    tol[..., at[0]] = 2 * U * ((a * c).abs() + (b * s).abs()) + U * y[..., at[0]].abs()
    tol[..., at[1]] = 2 * U * ((b * c).abs() + (a * s).abs()) + U * y[..., at[1]].abs()
    return y, tol


def check(got, x, cos, sin, positions, interleaved, inverse=False):
    want, tol = exact(x, cos, sin, positions, interleaved, inverse)
    step = 2.0 ** -8 if got.dtype == BF16 else 0.0
    off = (got.double() - want).abs()
    assert bool((off <= tol + step * (want.abs() + tol)).all()), float((off - tol).max())


def order(b, s, pos0=0):
    return (torch.arange(s, device=DEV) + pos0).expand(b, s).contiguous()


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dst", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("dim,half", [(64, 32), (128, 32), (80, 8), (50, 25), (2, 1), (7, 2), (256, 128), (96, 47)])
def test_shapes_and_types(dim, half, src, dst, interleaved, inverse):
    b, s, heads, kv = 2, 37, 5, 2
    cos, sin = tables(64, half)
    xs = rand(b, s, heads, dim, dtype=src), rand(b, s, kv, dim, dtype=src, seed=2)
    positions = (order(b, s) * 3 + 5 * order(s, b).t()) % 64
    flat = [torch.full((x.numel() + 33,), 7.0, dtype=dst, device=DEV) for x in xs]
    ys = [f[1:1 + x.numel()].view(x.shape) for f, x in zip(flat, xs)]
    P.rotary(xs, ys, cos, sin, positions.contiguous(), interleaved=interleaved, inverse=inverse)
    for x, y, f in zip(xs, ys, flat):
        check(y, x, cos, sin, positions, interleaved, inverse)
        assert bool((f[0] == 7.0)) and bool((f[1 + x.numel():] == 7.0).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,heads,dim", [(1, 1, 32, 128), (1, 1, 1, 4), (3, 1, 130, 256), (1, 9, 130, 256),
                                           (1, 70000, 1, 64), (2, 8192, 12, 64), (1, 3, 600, 64), (65, 33, 3, 36)])
def test_sizes(b, s, heads, dim, interleaved):
    """One token, tokens with more pieces than a workgroup takes, long sequences, either
    number of items a thread."""
    cos, sin = tables(s + 2, dim // 2 // 2)
    x = rand(b, s, heads, dim, dtype=BF16)
    y = torch.empty_like(x)
    P.rotary(x, y, cos, sin, pos0=2, interleaved=interleaved)
    check(y, x, cos, sin, order(b, s, 2), interleaved)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_views(interleaved, dtype):
    """Parts of a fused projection, heads before tokens, a sequence shared by the batch,
    every other token."""
    cos, sin = tables(100, 24)
    fused = rand(2, 21, 7, 64, dtype=dtype)
    heads_first = rand(2, 4, 21, 64, dtype=dtype, seed=3).transpose(1, 2)
    shared = rand(1, 21, 2, 64, dtype=dtype, seed=4).expand(2, 21, 2, 64)
    skipping = rand(2, 42, 3, 64, dtype=dtype, seed=5)[:, ::2]
    xs = (fused[:, :, :4], heads_first, shared, skipping)
    outs = torch.full((2, 21, 9, 64), 7.0, dtype=dtype, device=DEV)
    ys = (outs[:, :, 5:9], torch.empty(2, 4, 21, 64, dtype=dtype, device=DEV).transpose(1, 2),
          torch.empty(2, 21, 2, 64, dtype=dtype, device=DEV), outs[:, :, 1:4])
    positions = order(2, 21, 11)
    P.rotary(xs, ys, cos, sin, positions, interleaved=interleaved)
    for x, y in zip(xs, ys):
        check(y, x, cos, sin, positions, interleaved)
    assert bool((outs[:, :, 0] == 7.0).all()) and bool((outs[:, :, 4] == 7.0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place(interleaved, dtype):
    """q and k within their fused projection, v and the values behind the turned ones as
    they were; turned back they are what they were up to two roundings."""
    cos, sin = tables(90, 20)
    fused = rand(3, 30, 8, 72, dtype=dtype)
    was = fused.clone()
    views = (fused[:, :, :5], fused[:, :, 5:7])
    positions = order(3, 30, 60)
    P.rotary(views, views, cos, sin, positions, interleaved=interleaved)
    check(views[0], was[:, :, :5], cos, sin, positions, interleaved)
    check(views[1], was[:, :, 5:7], cos, sin, positions, interleaved)
    assert torch.equal(fused[:, :, 7], was[:, :, 7]) and torch.equal(fused[..., 40:], was[..., 40:])
    P.rotary(views, views, cos, sin, positions, interleaved=interleaved, inverse=True)
    step = 2.0 ** -8 if dtype == BF16 else 4 * U
    size = was[:, :, :7].double().abs().amax(-1, keepdim=True) * 2
    assert bool(((fused[:, :, :7].double() - was[:, :, :7].double()).abs() <= 4 * step * size).all())


def test_positions_that_the_table_does_not_hold():
    cos, sin = tables(10, 8)
    x = rand(1, 6, 2, 20)
    positions = torch.tensor([[0, 9, 10, -1, 2 ** 40, 3]], device=DEV)
    y = torch.empty_like(x)
    P.rotary(x, y, cos, sin, positions)
    good = [0, 1, 5]
    check(y[:, good], x[:, good], cos, sin, positions[:, good], False)
    assert bool(torch.isnan(y[:, 2:5, :, :16]).all()) and torch.equal(y[..., 16:], x[..., 16:])


def test_values_that_are_not_finite_stay_in_their_pair():
    cos, sin = tables(10, 8)
    for interleaved in (False, True):
        x = rand(1, 5, 2, 16)
        clean = x.clone()
        x[0, 2, 1, 3] = float("nan")
        y, z = torch.empty_like(x), torch.empty_like(x)
        P.rotary(x, y, cos, sin, interleaved=interleaved)
        P.rotary(clean, z, cos, sin, interleaved=interleaved)
        pair = (2, 3) if interleaved else (3, 11)
        bad = torch.isnan(y)
        assert int(bad.sum()) == 2 and all(bool(bad[0, 2, 1, i]) for i in pair)
        assert torch.equal(y[~bad], z[~bad])


def test_offsets_past_32_bits():
    """Tokens 2^31 values apart."""
    apart = (1 << 31) + 16
    big = torch.empty(apart + 64, dtype=BF16, device=DEV)
    x = big.as_strided((1, 2, 1, 64), (2 * apart, apart, 64, 1))
    small = rand(1, 2, 1, 64, dtype=BF16)
    x.copy_(small)
    cos, sin = tables(4, 32)
    y = torch.empty_like(small)
    P.rotary(x, y, cos, sin)
    check(y, small, cos, sin, order(1, 2), False)
    P.rotary(x, x, cos, sin)
    assert torch.equal(x.contiguous(), y)


def test_equals_the_prologue():
    """The whole head, half layout, in order: the fused prologue's values to a rounding of
    each product and sum."""
    rope = D.DeviceRope(RopeCache(64, 50, 1e4), pos0=7)
    q, k = rand(2, 40, 6, 64), rand(2, 40, 2, 64, seed=2)
    want = D.prologue_fwd(q, k, rope)[:2]
    got = A.rotary((q, k), rope.cos, rope.sin, pos0=7)
    for x, g, w in zip((q, k), got, want):
        check(g, x, rope.cos, rope.sin, order(2, 40, 7), False)
        check(w, x, rope.cos, rope.sin, order(2, 40, 7), False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_autograd(interleaved, dtype):
    """The gradient is the inverse turn: of the scaled table's transpose, so <y, g> = <x, dx>."""
    rope = RopeCache(24, 64, 1e4, YarnScaling(4.0, 16))
    cos, sin = (torch.from_numpy(t).to(DEV) for t in (rope.cos, rope.sin))
    q = rand(2, 17, 4, 40, dtype=dtype).requires_grad_()
    k = rand(2, 17, 2, 40, dtype=dtype, seed=2).transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    positions = (order(2, 17) * 2 + 9).contiguous()
    ys = A.rotary((q, k), cos, sin, positions, interleaved=interleaved, dtype=F32)
    assert all(y.dtype == F32 for y in ys)
    gs = rand(2, 17, 4, 40, seed=5), rand(2, 17, 2, 40, seed=6)
    grads = torch.autograd.grad(ys, (q, k), gs, retain_graph=True)
    for x, y, g, dx in zip((q, k), ys, gs, grads):
        check(y.detach(), x.detach(), cos, sin, positions, interleaved)
        assert dx.dtype == dtype
        check(dx, g, cos, sin, positions, interleaved, True)
    # One output that nothing depends on, and an expanded gradient.
    dq, dk = torch.autograd.grad(ys[0].sum(), (q, k))
    check(dq, torch.ones(2, 17, 4, 40, device=DEV), cos, sin, positions, interleaved, True)
    assert not dk.any()
    # Along a direction: the map is linear, so the difference is the derivative but for roundings.
    v = rand(2, 17, 4, 40, seed=7).to(dtype)
    lo = A.rotary((q.detach() - v), cos, sin, positions, interleaved=interleaved, dtype=F32)
    hi = A.rotary((q.detach() + v), cos, sin, positions, interleaved=interleaved, dtype=F32)
    step = (q.detach() + v).double() - (q.detach() - v).double()
    slope = float(((hi.double() - lo.double()) * gs[0]).sum())
    want = float((exact(gs[0], cos, sin, positions, interleaved, True)[0] * step).sum())
    room = 8 * U * float(((q.detach().double().abs() + v.double().abs()).amax() * 2 * 1.2 * gs[0].double().abs()).sum())
    assert abs(slope - want) <= room


def test_captured_replays():
    cos, sin = tables(300, 16)
    x = rand(2, 150, 5, 64)
    y = torch.empty_like(x)
    P.rotary(x, y, cos, sin)
    torch.cuda.synchronize()
    want = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.rotary(x, y, cos, sin)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        P.rotary(rand(1, 9, 3, 64), torch.empty(1, 9, 3, 64, device=DEV), cos, sin)
        torch.cuda.synchronize()


def test_empty():
    cos, sin = tables(10, 8)
    for shape in ((0, 5, 2, 16), (2, 0, 2, 16), (2, 5, 0, 16)):
        x = torch.empty(shape, device=DEV)
        P.rotary(x, torch.empty_like(x), cos, sin)
    x, none = rand(1, 5, 2, 16), torch.empty(1, 5, 0, 16, device=DEV)
    y = torch.empty_like(x)
    P.rotary((none, x, none), (none.clone(), y, none.clone()), cos, sin)
    check(y, x, cos, sin, order(1, 5), False)


def test_refusals():
    cos, sin = tables(10, 8)
    x = rand(1, 5, 2, 16)
    y = torch.empty_like(x)
    for kw, error in ((dict(pos0=6), ShapeError), (dict(pos0=-1), ValueError),
                      (dict(positions=torch.zeros(1, 5, dtype=torch.int32, device=DEV)), TypeError),
                      (dict(positions=torch.zeros(1, 4, dtype=torch.int64, device=DEV)), ShapeError)):
        with pytest.raises(error):
            P.rotary(x, y, cos, sin, **kw)
    big = tables(10, 9)
    for args, error in (((x, y, *big), ShapeError), ((x, y[:, :4], cos, sin), ShapeError),
                        ((x[0], y[0], cos, sin), ShapeError), ((x.cpu(), y, cos, sin), TypeError),
                        ((x.half(), y, cos, sin), TypeError), ((x, y, cos, sin[:9]), ShapeError),
                        ((x, y, cos, sin.t().contiguous()), ShapeError),
                        ((x, y, cos[0], sin[0]), ShapeError), ((x, y, cos.double(), sin), TypeError),
                        ((x.transpose(2, 3), y.transpose(2, 3), cos[:, :1].contiguous(), sin[:, :1].contiguous()),
                         ValueError),
                        ((x, torch.empty(1, 1, 2, 16, device=DEV).expand(1, 5, 2, 16), cos, sin), ValueError),
                        (((x, x), (y,), cos, sin), ValueError), (((x,) * 5, (y,) * 5, cos, sin), ValueError),
                        (((x, x.bfloat16()), (y, y.clone()), cos, sin), TypeError),
                        (((x, rand(1, 4, 2, 16)), (y, rand(1, 4, 2, 16)), cos, sin), ShapeError)):
        with pytest.raises(error):
            P.rotary(*args)
    # In place over other strides.
    with pytest.raises(CfattnError, match="in place"):
        flat = rand(4 * 16)
        P.rotary(flat.as_strided((1, 2, 2, 16), (64, 32, 16, 1)), flat.as_strided((1, 2, 2, 16), (64, 16, 32, 1)), cos,
                 sin)
