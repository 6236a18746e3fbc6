"""Attention and its gradient in float32 with products of several makings, and their errors against 64 bits."""
import numpy as np


def planes(x, count):
    """`x` as a sum of bfloat16 numbers (rounded to nearest, ties to even), each of what the ones before leave."""
    parts = []
    for _ in range(count):
        bits = x.astype(np.float32).view(np.uint32).astype(np.uint64)
        high = ((bits + 0x7fff + (bits >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
        parts.append(high)
        x = x - high
    return parts


def split_product(count):
    """Products of `count` bfloat16 parts of each operand, the small ones first: those of parts n and m with n + m < count."""
    def product(a, b):
        a, b = planes(a, count), planes(b, count)
        total = np.float32(0)
        for n, m in sorted(((n, m) for n in range(count) for m in range(count) if n + m < count), key=lambda p: -sum(p)):
            total = total + a[n] @ b[m]
        return total
    return product


def plain_product(a, b):
    return a @ b


def attention(q, k, v, g, product, kind=np.float32):
    """{o, dq, dk, dv} of one head without a mask."""
    q, k, v, g = (x.astype(kind) for x in (q, k, v, g))
    scale = kind(1.0 / np.sqrt(q.shape[1]))
    z = product(q * scale, k.T.copy())
    e = np.exp(z - z.max(1, keepdims=True))
    w = e / e.sum(1, keepdims=True, dtype=kind)
    o = product(w, v)
    ds = w * (product(g, v.T.copy()) - (g * o).sum(1, keepdims=True, dtype=kind)) * scale
    return {"o": o, "dq": product(ds, k), "dk": product(ds.T.copy(), q), "dv": product(w.T.copy(), g)}


def error(got, want):
    """Root mean square error, in parts of the result's root mean square."""
    return np.sqrt(((got.astype(np.float64) - want) ** 2).mean() / (want ** 2).mean())


# A sum of float32 numbers is off by about sqrt(n) half steps after n additions.  The plain products here add in
# vectors of 8 or 16 lanes, a matrix instruction in a chain: of 128 elements 48 additions (8 steps of 6 products) for 8 to
# 16, of n keys 6 n / 16 for n / 16 to n / 8: 2.5 times the error at most, with what the scores' errors bring to the
# weights 3 times.  Two parts instead of three leave out 2^-17 of an operand where float32 rounds off 2^-24.
WORST = 3.0
SIZES = [(96, 64, 128), (160, 700, 128), (130, 4096, 128), (200, 1000, 64)]


def inputs(lq, lk, d):
    rs = np.random.RandomState(lq + lk)
    return [rs.standard_normal((n, d)).astype(np.float32) for n in (lq, lk, lk, lq)]
