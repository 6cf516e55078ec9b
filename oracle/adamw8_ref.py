"""AdamW with 8-bit moments on the CPU: the format and its stochastic rounding in integer and fp64 arithmetic (exact), the
moments in single-rounded fp32 operations as defined, the parameters in fp64."""
import numpy as np

BLOCK = 64
TOP = {True: 15, False: 31}                    # exponent field of the block's scale: signed first moment, second moment
NEAREST = 1 << 19


def dither(n, seed, step):
    """The two dithers of elements 0..n-1 of a tensor, in units of 2^-20 code steps: the middles of 2^16 equal parts."""
    m64 = 2 ** 64 - 1
    key = (seed % 2 ** 64 * 0x9E3779B97F4A7C15 + step * 0x6A09E667F3BCC909) & m64
    key = (((key ^ (key >> 31)) * 0x9E3779B97F4A7C15) & m64) >> 32
    i = np.arange(n, dtype=np.uint64)
    h = ((i & np.uint64(0xffffffff)) * np.uint64(0x9E3779B9) + (i >> np.uint64(32)) * np.uint64(0xBB67AE85) + np.uint64(key)) & np.uint64(0xffffffff)
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0x6A09E667)) & np.uint64(0xffffffff)
    h = (h ^ (h >> np.uint64(16))).astype(np.int64)
    return ((h & 0xffff) << 4) | 8, ((h >> 16) << 4) | 8


def exponents(x):
    """Per block of 64 of fp32 x (the last one may be short)."""
    bits = (x.astype(np.float32).view(np.int32) & 0x7fffffff).astype(np.int64)
    pad = np.zeros(-len(x) % BLOCK, np.int64)
    e = (np.concatenate([bits, pad]).reshape(-1, BLOCK).max(1) + 0xfffff) >> 23
    return np.clip(e, 32, 255)


def encode(x, signed, d):
    """-> (codes, exponents): |x| in units of the smallest code, plus d / 2^20, rounded down."""
    e = exponents(x)
    per = np.repeat(e, BLOCK)[:len(x)]
    ok = per < 255
    top = TOP[signed]
    mag = np.where(ok, np.abs(x.astype(np.float64)), 0.0)
    y = np.ldexp(mag, (127 + top + 2 - per).astype(np.int64))         # in units of the smallest code, 2^(e - 127 - top - 2)
    y = np.where(y < 8, np.rint(y * 2.0 ** 20) / 2.0 ** 20, y)        # below the normal range 20 bits of fraction are kept
    field = np.maximum(np.floor(np.log2(np.maximum(y, 8.0))).astype(np.int64) - 3, 0)    # binade: the code steps by 2^field units
    frac = np.ldexp(y, -field) + d / 2.0 ** 20
    c = np.floor(frac).astype(np.int64) + 8 * field
    c = np.where(ok, c, 0)
    if signed:
        c = np.where(ok & (x < 0), c | 128, c)
    else:
        c = np.where(ok & (x > 0) & (c == 0), 1, c)
    return c.astype(np.uint8), e.astype(np.uint8)


def decode(c, e, signed):
    """fp64 values (exact)."""
    per = np.repeat(e.astype(np.int64), BLOCK)[:len(c)]
    c = c.astype(np.int64)
    mag = c & 127 if signed else c
    field, frac = np.maximum(mag >> 3, 1), np.where(mag >= 8, 8 + (mag & 7), mag)
    v = np.ldexp(frac.astype(np.float64), field - 1 + per - 127 - TOP[signed] - 2)
    v = np.where((c >= 128) & signed, -v, v)
    return np.where(per == 255, np.nan, v)


def step(p, g, m8, v8, coef, lr, b1, b2, eps, wd, t, seed):
    """One tensor; m8, v8 = (codes, exponents).  -> (p in fp64, bound on an fp32 p, m8, v8)."""
    f = np.float32
    with np.errstate(all="ignore"):
        g = (g.astype(f) * f(coef)).astype(f)
        m0, v0 = decode(*m8, True).astype(f), decode(*v8, False).astype(f)
        m = m0 + (g - m0) * f(1 - b1)
        v = v0 * f(b2) + (f(1 - b2) * g) * g
        assert m.dtype == v.dtype == np.float32
        # the parameters from the same moments in fp64
        denom = np.sqrt(v.astype(np.float64)) / np.sqrt(1 - b2 ** t) + eps
        upd = lr / (1 - b1 ** t) * m.astype(np.float64) / denom
        p64 = p.astype(np.float64) * (1 - lr * wd)
        u = 2.0 ** -24
        # decay and its product 2, sum 1; root, its factor, sum, quotient, size and product: 8, with 4 to spare for a root
        # and a quotient that are a unit in the last place off instead of half a one
        bound = 3 * u * np.abs(p64) + (12 + 1) * u * np.abs(upd)
        dm, dv = dither(len(p), seed, t)
        return p64 - upd, bound, encode(m, True, dm), encode(v, False, dv)
