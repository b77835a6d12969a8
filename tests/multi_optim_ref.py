"""Plain restatements of the many-tensor optimizer operators for the tests: numpy, 64 bits, and for the 8-bit codes integer
arithmetic on levels (mantissa and exponent), written from the definition."""
import numpy as np

EPS24 = 2.0 ** -24          # half a step of fp32, relative
BLOCK = 256
A, RATE_M, RATE_V = 0x9E3779B9, 0xBB67AE85, 0x6A09E667


def norm(grads):
    return float(np.sqrt(sum(float(np.sum(np.asarray(g, np.float64) ** 2)) for g in grads)))


def coefficient(n, max_norm):
    return min(1.0, max_norm / (n + 1e-6))


def adamw(p, g, m, v, t, lr=1e-4, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, coef=1.0):
    """step t in 64 bits: (p, m, v) and a bound on each one's error in fp32 arithmetic.  Roundings counted per operation, half a step each:
    m: coef, coef g, the constants' own rounding (2), two products, the sum: at most 6 halves of |b1 m| + |(1 - b1) g|.
    v: the same with g squared (coef and coef g count twice, one product more): 10 halves.
    the step: lr and the bias corrections rounded (2), product, root, its factor, sum with eps (rounded itself), division: 8 halves.
    With 8-bit moments root and reciprocal are the hardware's, off by a whole last place each (2 halves instead of 1, the reciprocal's
    product 1 more; root's factor and sum are one operation, 1 less): step size, product, 2 root + factor rounded, sum, 2 + 1: 9 halves.
    Plus m's error over the divisor and half of v's relative error (5 halves): 14; then decay (2), product and difference of p."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    g = g * coef
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    dm = 6 * EPS24 * (np.abs(b1 * m) + np.abs((1 - b1) * g))
    dv = 10 * EPS24 * v1
    den = np.sqrt(v1) / np.sqrt(1 - b2 ** t) + eps
    step = lr / (1 - b1 ** t) * m1 / den
    p1 = p * (1 - lr * wd) - step
    dp = EPS24 * (3 * np.abs(p) + np.abs(p1) + 14 * np.abs(step)) + lr / (1 - b1 ** t) * dm / den
    return (p1, m1, v1), (dp, dm, dv)


def moments32(g, m, v, b1=0.9, b2=0.999):
    """m and v of a step in fp32, one rounding per operation, in the kernel's order: the same bits"""
    f = np.float32
    g, m, v = (np.asarray(x, f) for x in (g, m, v))
    with np.errstate(all="ignore"):
        return f(b1) * m + f(1 - b1) * g, f(b2) * v + f(1 - b2) * g * g


def dither(n, t, rate):
    return (((np.arange(n, dtype=np.uint64) * A + np.uint64(t * rate % 2 ** 32)) & np.uint64(0xFFFFFFFF)) >> np.uint64(12)).astype(np.int64)


def _levels(x):
    """exact: x = value(level) * (1 + part / (8 + level % 8)); zero has no level.  fp32's level numbers: 8 * 127 is 1.0"""
    frac, e = np.frexp(x)
    y = frac * 16
    lo = np.floor(y)
    return 8 * (e.astype(np.int64) + 126) + lo.astype(np.int64) - 8, y - lo


def level_value(level):
    level = np.asarray(level, np.int64)
    return np.ldexp((8 + level % 8) / 16.0, level // 8 - 126)


def pack(x, d, codes, signed):
    """codes and base of ONE block's values (normal fp32 numbers, zeros, NaN, infinities); d: dither of each, in [0, 2^20)"""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x)
    a = np.where(fine, np.abs(x), 0.0)
    some = a > 0
    lev, part = _levels(np.where(some, a, 1.0))
    top = max([int(l + (q > 0)) for l, q in zip(lev[some], part[some])], default=0)
    base = max(min(top, 0x7F7) - codes, 0)
    c = lev + (part * 2 ** 20 + d >= 2 ** 20) - base
    if signed:
        low = level_value(base + 1)
        c = np.where(a >= low, np.minimum(c, codes), (a > d * (low / 2 ** 20)).astype(np.int64))
    else:
        c = np.clip(c, 1, codes)
    c = np.where(some, c, 0)
    if signed:
        q = np.where(c > 0, c + 128 * (x < 0), 0)
        return np.where(fine, q, 128).astype(np.uint8), base
    return np.where(fine, c, 255).astype(np.uint8), base


def unpack(q, base, signed):
    q = np.asarray(q, np.int64)
    c = q & 127 if signed else q
    x = np.where(c > 0, level_value(base + c), 0.0)
    if signed:
        return np.where(q == 128, np.nan, np.where(q > 128, -x, x))
    return np.where(q == 255, np.nan, x)


def pack_tensor(x, t, rate, codes, signed, nearest=False):
    """all blocks of one tensor: (codes, bases)"""
    x = np.asarray(x).reshape(-1)
    d = np.full(x.size, 1 << 19, np.int64) if nearest else dither(x.size, t, rate)
    q, bases = np.zeros(x.size, np.uint8), []
    for b in range(0, x.size, BLOCK):
        q[b:b + BLOCK], base = pack(x[b:b + BLOCK], d[b:b + BLOCK], codes, signed)
        bases.append(base)
    return q, np.array(bases, np.int64)


def unpack_tensor(q, bases, signed):
    q = np.asarray(q).reshape(-1)
    return np.concatenate([unpack(q[b:b + BLOCK], int(bases[b // BLOCK]), signed) for b in range(0, q.size, BLOCK)] or [np.zeros(0)])
