"""GPU tests of AdamW with 8-bit moments (cfops_adamw8_*) against its numpy
restatement in 64 bits (tests/adamw8_ref.py)."""
import numpy as np
import pytest
import torch

from cpuforge_amd import _lib
from tests import adamw8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HP = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(DEV)


def inputs(n, seed, spread=2.0):
    """p, g, m, v; sizes that spread over e^spread by value, moments as held."""
    r = np.random.RandomState(seed)
    size = np.exp(r.standard_normal(n) * spread)
    p, g, m, v = r.standard_normal(n), r.standard_normal(n) * size, r.standard_normal(n) * size, (r.randn(n) * size) ** 2
    p, g, m, v = (x.astype(np.float32).astype(np.float64) for x in (p, g, m, v))
    half = np.full(n, 0.5)
    return p, g, R.held(m, R.LEAST_M, half), R.held(v, R.LEAST_V, half, positive=True)


def table(p, g, m, v, wd, off=0):
    from cpuforge_amd import ops as P
    n = p.size
    d = {}
    for k, x in dict(p=p, g=g, m=m, v=v).items():
        d[k] = torch.empty(n + off, device=DEV)[off:]
        d[k].copy_(dev(x))
    d["state8"] = P.adamw8_state(n, DEV)
    d["weight_decay"] = wd
    return d


def moments(d):
    from cpuforge_amd import ops as P
    out = dict(d, m=torch.full_like(d["m"], -7.0), v=torch.full_like(d["v"], -7.0))
    P.adamw8_unpack_multi([out])
    return out["m"].cpu().numpy().astype(np.float64), out["v"].cpu().numpy().astype(np.float64)


def assert_step(got_p, want_p, p, g, m, v, t, wd):
    """p to f32: its own rounding, and the update's: five roundings and the
    library's square root and quotient (two more), on lr * update."""
    upd = np.abs(want_p - p)
    tol = 2.0 ** -24 * np.abs(want_p) + 10 * 2.0 ** -24 * (upd + HP["lr"] * wd * np.abs(p)) + 1e-45
    assert (np.abs(got_p - want_p) <= tol).all(), np.abs(got_p - want_p).max()


@pytest.mark.parametrize("n,off", [(1, 0), (3, 1), (255, 0), (256, 0), (257, 2), (4095, 0), (4096, 0), (4097, 3),
                                   (70001, 0), (70001, 1)])
def test_steps_match_64_bits(n, off):
    from cpuforge_amd import ops as P
    print(n, off, flush=True)
    p, g, m, v = inputs(n, n + off)
    d = table(p, g, m, v, 0.1, off)
    P.adamw8_pack_multi([d])
    m0, v0 = moments(d)
    assert np.array_equal(m0, m) and np.array_equal(v0, v)  # held values are held
    for t in (3, 4, 5):
        p1, m1, v1 = R.step(p, g, m, v, t, HP["lr"], HP["beta1"], HP["beta2"], HP["eps"], 0.1)
        P.adamw8_update_multi([d], t, **HP)
        got = d["p"].cpu().numpy().astype(np.float64)
        assert_step(got, p1, p, g, m, v, t, 0.1)
        gm, gv = moments(d)
        # The same side of every threshold: a sum rounded in 53 bits against
        # another order's, and a threshold of 17 bits.
        assert np.array_equal(gm, m1) and np.array_equal(gv, v1)
        p, m, v = got, gm, gv


def test_nothing_behind_a_tensor_is_written():
    from cpuforge_amd import ops as P
    n = 300
    p, g, m, v = inputs(n, 5)
    big = {k: torch.full((n + 64,), 3.0, device=DEV) for k in "pgmv"}
    for k, x in dict(p=p, g=g, m=m, v=v).items():
        big[k][:n] = dev(x)
    room = torch.full((P.adamw8_state(n, DEV).numel() + 64,), 9, dtype=torch.uint8, device=DEV)
    d = {k: big[k][:n] for k in "pgmv"} | dict(state8=room[:-64], weight_decay=0.0)
    P.adamw8_pack_multi([d])
    P.adamw8_update_multi([d], 1, **HP)
    P.adamw8_unpack_multi([d])
    assert all(bool((big[k][n:] == 3.0).all()) for k in "pgmv") and bool((room[-64:] == 9).all())


@pytest.mark.parametrize("count", [1, 16, 17, 60, 447, 448, 449, 700])
def test_mixed_tensors(count):
    """8-bit and 32-bit states in one call; the 32-bit ones are bit for bit
    adamw_update's, empty tensors are passed over."""
    from cpuforge_amd import ops as P
    sizes = [1, 4096, 0, 4097, 8191, 576, 12289]
    ts, want = [], []
    for i in range(count):
        n = sizes[i % len(sizes)]
        p, g, m, v = inputs(n, i) if n else (np.zeros(0),) * 4
        d = table(p, g, m, v, 0.1 * (i % 2), i % 5 % 3)
        one = {k: x.clone() for k, x in d.items() if k in "pgmv"}
        if i % 3 == 1:
            del d["state8"]
            P.adamw_update(one["p"], one["g"], one["m"], one["v"], 2, 1e-2, 0.9, 0.99, 1e-8, 0.1 * (i % 2))
        else:
            one.update(state8=torch.zeros_like(d["state8"]), weight_decay=d["weight_decay"])
            P.adamw8_pack_multi([one])
            P.adamw8_update_multi([one], 2, **HP)
        ts.append(d)
        want.append(one)
    tab = P.Adamw8Tensors(ts)
    P.adamw8_pack_multi(tab)
    P.adamw8_update_multi(tab, 2, **HP)
    for d, one in zip(ts, want):
        for k in ("p", "state8") if "state8" in d else ("p", "m", "v"):
            assert torch.equal(d[k], one[k]), k


def test_tensors_that_share_memory_are_updated_in_order():
    from cpuforge_amd import ops as P
    p, g, m, v = inputs(9000, 3)
    a = table(p, g, m, v, 0.0)
    P.adamw8_pack_multi([a])
    b = {k: (x.clone() if isinstance(x, torch.Tensor) else x) for k, x in a.items()}
    P.adamw8_update_multi([a, a], 1, **HP)
    for _ in range(2):
        P.adamw8_update_multi([b], 1, **HP)
    assert torch.equal(a["p"], b["p"]) and torch.equal(a["state8"], b["state8"])


def test_odd_gradients():
    """NaN and infinite gradients poison their own value alone.  (The square of
    3e19 times 1 - beta2 is 9e36, which f32 holds.)"""
    from cpuforge_amd import ops as P
    n = 600
    p, g, m, v = inputs(n, 9)
    g[[5, 300]] = np.nan
    g[6] = np.inf
    g[301] = 3e19
    d = table(p, g, m, v, 0.0)
    P.adamw8_pack_multi([d])
    ok = np.ones(n, bool)
    ok[[5, 6, 300]] = False
    p1, m1, v1 = R.step(p, g, m, v, 1, HP["lr"], HP["beta1"], HP["beta2"], HP["eps"], 0.0)
    P.adamw8_update_multi([d], 1, **HP)
    got = d["p"].cpu().numpy().astype(np.float64)
    gm, gv = moments(d)
    assert np.array_equal(np.isnan(got), ~ok)
    assert np.array_equal(np.isfinite(gm), ok) and np.array_equal(np.isinf(gv), ~ok)
    assert np.array_equal(gm[ok], m1[ok]) and np.array_equal(gv[ok], v1[ok])
    P.adamw8_update_multi([d], 2, **HP)  # and the poison stays where it is
    assert np.array_equal(np.isfinite(d["p"].cpu().numpy()), ok)


def test_a_square_that_f32_does_not_hold():
    """stops its value's update, as with 32-bit states."""
    from cpuforge_amd import ops as P
    n = 600
    p, g, m, v = inputs(n, 10)
    g[301] = 3e20
    d = table(p, g, m, v, 0.0)
    P.adamw8_pack_multi([d])
    _, m1, v1 = R.step(p, g, m, v, 1, HP["lr"], HP["beta1"], HP["beta2"], HP["eps"], 0.0)
    P.adamw8_update_multi([d], 1, **HP)
    gm, gv = moments(d)
    assert np.array_equal(gm, m1) and np.array_equal(gv, v1) and np.isinf(gv[301]) and np.isinf(gv).sum() == 1
    for t in (2, 3):
        assert float(d["p"][301]) == np.float32(p[301])
        P.adamw8_update_multi([d], t, **HP)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-42, 1e17])
def test_extreme_blocks(scale):
    from cpuforge_amd import ops as P
    n = 512
    p, g, m, v = inputs(n, 11)
    g, m = (np.float32(x * scale).astype(np.float64) for x in (g, m))
    v = np.float32(np.minimum(v * scale * scale, 1e38)).astype(np.float64)
    half = np.full(n, 0.5)
    m, v = R.held(m, R.LEAST_M, half), R.held(v, R.LEAST_V, half, positive=True)
    d = table(p, g, m, v, 0.0)
    P.adamw8_pack_multi([d])
    gm, gv = moments(d)
    # (f32 rounds what lies below its least normal.)
    assert np.abs(gm - m).max() <= 2.0 ** -150 and np.abs(gv - v).max() <= 2.0 ** -150
    P.adamw8_update_multi([d], 1, **HP)
    assert bool(torch.isfinite(d["p"]).all())
    if scale == 0.0:
        gm, gv = moments(d)  # (zeros, some of them negative)
        same = np.array_equal(d["p"].cpu().numpy(), p.astype(np.float32))
        assert same and not gm.any() and not gv.any()


def test_replayed_steps_equal_eager_ones():
    """A captured step replayed, with eager work between (its step count is the
    captured one's)."""
    from cpuforge_amd import ops as P
    p, g, m, v = inputs(50000, 13)
    a = table(p, g, m, v, 0.1)
    P.adamw8_pack_multi([a])
    b = {k: (x.clone() if isinstance(x, torch.Tensor) else x) for k, x in a.items()}
    ta, tb = P.Adamw8Tensors([a]), P.Adamw8Tensors([b])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            P.adamw8_update_multi(ta, 4, **HP)
    torch.cuda.synchronize()
    for i in range(4):
        graph.replay()
        P.adamw8_update_multi(tb, 4, **HP)
        torch.cuda.synchronize()
        assert torch.equal(a["p"], b["p"]) and torch.equal(a["state8"], b["state8"]), i


def test_refusals():
    from cpuforge_amd import ops as P
    x = torch.zeros(300, device=DEV)
    s = P.adamw8_state(300, DEV)
    with pytest.raises(_lib.ShapeError):
        P.Adamw8Tensors([dict(p=x, g=x, state8=s[:-1])])
    with pytest.raises(_lib.ShapeError):
        P.Adamw8Tensors([dict(p=x, g=x[:5], state8=s)])
    with pytest.raises(TypeError):
        P.Adamw8Tensors([dict(p=x, g=x, state8=x)])
    with pytest.raises(_lib.CfattnError, match="aligned"):
        big = torch.zeros(s.numel() + 1, dtype=torch.uint8, device=DEV)
        P.adamw8_update_multi([dict(p=x, g=x, state8=big[1:])], 1, **HP)
    with pytest.raises(_lib.CfattnError, match="null"):
        P.adamw8_update_multi([dict(p=x, state8=s)], 1, **HP)
    with pytest.raises(_lib.CfattnError, match="null"):
        P.adamw8_unpack_multi([dict(p=x, g=x, state8=s)])


class Model:
    lora_cfg = None

    def __init__(self, named):
        self.named = named

    def named_params(self):
        return iter(self.named)


def model(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    named = []
    for name, shape in (("a.weight", (70, 100)), ("a.norm", (64,)), ("b.weight", (5, 9)), ("c.weight", (64, 64))):
        p = torch.randn(shape, generator=g, device=DEV).requires_grad_()
        named.append((name, p))
    return Model(named)


def set_grads(m, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    for _, p in m.named:
        p.grad = torch.randn(p.shape, generator=g, device=DEV)


def test_optimizer_with_8_bit_states_resumes(tmp_path):
    """Steps after a save and load equal the steps without one, bit for bit."""
    from cpuforge_amd.optim import AdamW, State8
    from cpuforge_amd.state import load_state, save_state
    m, opt = model(1), AdamW(0.9, 0.99, 1e-8, 0.1, state_bits=8)
    for i in range(5):
        set_grads(m, i)
        opt.update(m, 1e-2)
    assert isinstance(opt.state["a.weight"], State8) and isinstance(opt.state["a.norm"], tuple)
    save_state(tmp_path / "s.safetensors", m, opt, 5, 40)
    m2, opt2 = model(2), AdamW(0.9, 0.99, 1e-8, 0.1, state_bits=8)
    assert load_state(tmp_path / "s.safetensors", m2, opt2) == (5, 40)
    for i in range(5, 8):
        for a, o in ((m, opt), (m2, opt2)):
            set_grads(a, i)
            o.update(a, 1e-2)
    for (n, p), (_, q) in zip(m.named, m2.named):
        assert torch.equal(p, q), n
    # A file of 32-bit states goes on in 8, and the reverse.
    opt3 = AdamW(0.9, 0.99, 1e-8, 0.1)
    load_state(tmp_path / "s.safetensors", m2, opt3)
    set_grads(m2, 9)
    opt3.update(m2, 1e-2)
    assert isinstance(opt3.state["a.weight"], tuple)
    opt3.state["a.weight"] = State8.pack(*opt3.state["a.weight"])
    opt3.update(m2, 1e-2)
    assert isinstance(opt3.state["a.weight"], tuple)


def test_second_moment_follows_a_change_of_the_gradients():
    """beta2 = 0.999: v is to go from 1 to 1e-4 over 9000 steps and back; a v
    rounded to nearest would not move.  Held to a factor of two (a
    thousand-step mean of roundings of up to an eighth)."""
    from cpuforge_amd import ops as P
    n = 256
    d = table(np.zeros(n), np.full(n, 1e-2), np.zeros(n), np.ones(n), 0.0)
    P.adamw8_pack_multi([d])
    tab = P.Adamw8Tensors([d])
    for t in range(1, 9201):
        P.adamw8_update_multi(tab, t, 1e-6, 0.9, 0.999, 1e-8)
    _, v = moments(d)
    want = 0.999 ** 9200 + 1e-4 * (1 - 0.999 ** 9200)
    assert want / 2 < np.median(v) < want * 2, (np.median(v), want)
