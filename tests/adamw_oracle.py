"""Plain forms the optimizer tests compare with: the step in float64, and the 8-bit moments in elementary float32 operations (numpy),
each rounded once, which the kernel has to meet bit for bit."""
import numpy as np

BLOCK = 128
F = np.float32


def mix32(x):
    x = np.asarray(x, dtype=np.uint64) & 0xFFFFFFFF
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x21f0aaad)) & np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0x735a2d97)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(15))


def hashes(n, seed, index, step, first=0):
    """The 32-bit hash of elements first ... first + n - 1 of the tensor in place `index` of the list at step `step`."""
    key = mix32(int(mix32((step ^ seed) & 0xFFFFFFFF)) ^ ((seed >> 32) + index * 0x9e3779b9 & 0xFFFFFFFF))
    i = np.arange(first, first + n, dtype=np.uint64)
    return mix32((i & np.uint64(0xFFFFFFFF)) ^ mix32(np.uint64(key) ^ (i >> np.uint64(32))))


def decode(code, mantissa, bias):
    """float32 value of an 8-bit floating code (sign, 7 - mantissa exponent bits, mantissa); no infinities or NaN among them."""
    code = np.asarray(code, dtype=np.uint8).astype(np.int64)
    mag, e = code & 127, (code & 127) >> mantissa
    frac = (mag & ((1 << mantissa) - 1)) + np.where(e > 0, 1 << mantissa, 0)
    return (np.where(code > 127, -1., 1.) * np.ldexp(frac.astype(np.float64), np.maximum(e, 1) - bias - mantissa)).astype(F)


def blocks(x):
    n = x.size
    return np.concatenate([x, np.zeros(-n % BLOCK, dtype=x.dtype)]).reshape(-1, BLOCK)


def encode(x, r16, mantissa, bias, top):
    """(codes of |x| uint8, scales float32 [blocks]); x float32, r16 = 16 random bits per element."""
    with np.errstate(all='ignore'):
        big = np.abs(blocks(x)).max(1) if x.size else np.zeros(0, F)
        some = big >= F(2.0 ** -100)
        inv = np.where(some, F(1) / big * F(top), F(0)).astype(F)
        t = (np.abs(blocks(x)) * inv[:, None]).reshape(-1)[:x.size]
        e = np.maximum((t.view(np.int32) >> 23), 127 + 1 - bias)
        u = (r16.astype(F) + F(0.5)) * F(2.0 ** -16)
        k = np.floor(np.ldexp(t, mantissa + 127 - e).astype(F) + u).astype(np.int64)
    return (((e - (128 - bias)) << mantissa) + k).astype(np.int64), np.where(some, big * (F(1) / F(top)), F(0)).astype(F), t


def moments8(g, mc, vc, scales, factor, b1, b2, seed, index, step):
    """(exp_avg codes, exp_avg_sq codes, scales, m, v float32 unrounded) after one step from codes; g float32, all flat in memory order."""
    n = g.size
    sm, sv = (np.repeat(scales[:, j], BLOCK)[:n] for j in (0, 1))
    x = g * F(factor)
    m = F(b1) * (decode(mc, 3, 7) * sm) + F(1 - b1) * x
    v = F(b2) * (decode(vc, 2, 15) * sv) + F(1 - b2) * x * x
    h = hashes(n, seed, index, step)
    cm, ms, _ = encode(m, (h & np.uint64(0xFFFF)).astype(np.int64), 3, 7, 448.)
    cv, vs, tv = encode(v, (h >> np.uint64(16)).astype(np.int64), 2, 15, 57344.)
    cm = cm + np.where((cm > 0) & (m < 0), 128, 0)
    cv = np.maximum(cv, tv > 0)
    return cm.astype(np.uint8), cv.astype(np.uint8), np.stack([ms, vs], 1), m, v


def step64(p, g, m, v, t, lr, b1, b2, eps, wd, factor=1.0):
    """One step in float64 on float64 arrays; (p, m, v, and how far float32 may be off each: see `bounds`)."""
    x = g * factor
    m1, v1 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    size, denom = lr / (1 - b1 ** t), np.sqrt(v1 / (1 - b2 ** t)) + eps
    p1 = p * (1 - lr * wd) - size * m1 / denom
    # float32, u = 2^-24 a rounding: m: the difference x - m, its product, the sum and the constant: 4 u (|m| + |x|); v alike.
    # p: product with (1 - lr wd), its constant, the sum: 4 u |p|; the update: its factors (m, 1 / denom, sqrt, reciprocal of 1 ulp = 2 u,
    # step size, products) are at most 16 u off each other's size, with m's own error taken at |m| + |x|.
    u = 2.0 ** -24
    em, ev = 4 * u * (np.abs(m) + np.abs(x)), 4 * u * (v + x * x)
    ep = 4 * u * np.abs(p) + 16 * u * size * (np.abs(m) + np.abs(x)) / denom
    return p1, m1, v1, ep, em, ev
