"""AdamW with 8-bit moments restated in numpy, in 64 bits: the format, its
rounding and one step (include/cfops.h, cfops_adamw_tensor)."""
import numpy as np

BLOCK = 256
LEAST_M, LEAST_V = -13, -29  # the first normal binade, from the block's


def thresholds(n, t):
    """17 rounding bits of each of n values for m and for v at step t."""
    m32 = np.uint64(0xFFFFFFFF)

    def mix(x):
        x = ((x ^ (x >> np.uint64(16))) * np.uint64(0xA511E9B3)) & m32
        x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x63D83595)) & m32
        return x ^ (x >> np.uint64(16))
    key = mix(np.uint64((t * 0x9E3779B1 + 0x7F4A7C15) & 0xFFFFFFFF))
    h = mix((np.arange(n, dtype=np.uint64) + key) & m32)
    return (h & np.uint64(0x1FFFF)).astype(np.float64) / 2 ** 17, (h >> np.uint64(15)).astype(np.float64) / 2 ** 17


def blocks(x):
    """[blocks, 256] with zeros behind the last value."""
    out = np.zeros((-(-x.size // BLOCK), BLOCK))
    out.reshape(-1)[:x.size] = x.reshape(-1)
    return out


def exponent(a):
    """e of the block's (2^e, 2^(e+1)], to 2^-20, at least -127; of finite values."""
    big = np.where(np.isfinite(a), a, 0.0).max(1, keepdims=True)
    f, e = np.frexp(big)
    e = e - 1 - (2 * f < 1 + 2.0 ** -20)
    return np.where(big > 0, np.maximum(e, -127), -127).astype(np.float64)


def held(x, least, u, positive=False):
    """The values that 8 bits hold of x (1-d); u the thresholds in [0, 1)."""
    b, u = blocks(x), blocks(u)
    a = np.abs(b)
    e = exponent(a)
    with np.errstate(invalid="ignore", over="ignore"):
        lead = np.where((a > 0) & np.isfinite(a), np.frexp(a)[1] - 1.0, -400.0)
        step = np.exp2(np.maximum(lead, e + least) - 3)
        k = np.floor(a / step + u) * step
    if positive:
        k = np.where(a > 0, np.maximum(k, np.exp2(e + least - 3)), k)
    k = np.where(np.isfinite(a), k, np.inf if positive else np.nan)
    return np.copysign(k, b).reshape(-1)[:x.size]


def step(p, g, m, v, t, lr, beta1, beta2, eps, wd):
    """(p, m, v) after one step, m and v as held."""
    b1, b2, lr, eps, wd = (float(np.float32(x)) for x in (beta1, beta2, lr, eps, wd))
    with np.errstate(invalid="ignore", over="ignore"):
        m = b1 * m + float(np.float32(1) - np.float32(b1)) * g
        v = b2 * v + float(np.float32(1) - np.float32(b2)) * g * g
        m_in, v_in = (np.float32(x).astype(np.float64) for x in (m, v))  # what the update reads
        upd = m_in / (1 - b1 ** t) / (np.sqrt(v_in) / np.sqrt(1 - b2 ** t) + eps) + wd * p
        v = np.where(v < 2.0 ** 128, v, np.inf)
    um, uv = thresholds(p.size, t)
    return p - lr * upd, held(m, LEAST_M, um), held(v, LEAST_V, uv, positive=True)
