"""The oracle of the operators in `delayrepay_amd.nn`: their formulas head by head in float64, and
bounds for what float32 arithmetic may be off.

Bounds are of first order in u = 2^-24 (half a step of float32, relative): a sum of n products is off by
at most n u times the sum of their magnitudes, whatever its order, and an error of size e in a score is a
relative error of e in its weight.
"""
import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -125      # weights below the smallest normal number, 2^-126, may become zero: so much more is a weight off


def pairs(lq, lk, *, causal=False, start=None, length=None, prefix=0, documents=None):
    """(positions of the rows, whether row i sees key j) of one sequence."""
    n = lk if length is None else length
    start = n - lq if start is None else start
    p = start + np.arange(lq)
    ok = np.zeros((lq, lk), bool)
    for i in range(lq):
        for j in range(n):
            see = not causal or j <= p[i] or j < prefix
            if documents is not None:
                see = see and 0 <= p[i] < n and documents[p[i]] == documents[j]
            ok[i, j] = see
    return p, ok


def head(q, k, v, p, ok, scale, cap=None, slope=None, dout=None):
    """One head: dict of o, lse and their bounds, with `dout` of dq, dk, dv too.  Keys that no row sees
    count as zeros, so that they may hold anything."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    seen = ok.any(0)
    k, v = np.where(seen[:, None], k, 0.0), np.where(seen[:, None], v, 0.0)
    row = ok.any(1)
    q = np.where(row[:, None], q, 0.0)
    d, n = q.shape[1], k.shape[0]
    x = q @ k.T * scale
    t = np.zeros_like(x)
    # a product of d terms, the scaling, the change to units of log 2 and back
    size = np.abs(q) @ np.abs(k).T * abs(scale)
    off = (d + 6) * U * size
    z, zsize = x, np.abs(x)
    if cap is not None:
        t = np.tanh(x / cap)
        z = cap * t
        off = off + 6 * U * np.abs(z)        # (the slope of tanh is at most 1)
        zsize = np.abs(z)
    if slope is not None:
        far = slope * np.abs(p[:, None] - np.arange(n))
        z = z - far
        off = off + 4 * U * np.abs(far)
        zsize = zsize + np.abs(far)
    off = off + 4 * U * zsize                # the rounding of the score and of its distance to the largest
    z = np.where(ok, z, -np.inf)
    top = np.where(row, z.max(1, initial=-np.inf), 0.0)[:, None]
    e = np.where(ok, np.exp(z - top), 0.0)
    total = e.sum(1, keepdims=True)
    w = e / np.where(total == 0, 1.0, total)
    worst = np.where(ok, off, 0.0).max(1, initial=0.0)[:, None]
    # weight: its score, the largest's, the exponential (2 u), the sum (its terms' errors and n u), the quotient
    rel = off + 2 * worst + (n + 16) * U
    o = w @ v
    got = {"o": o, "o_off": (w * (rel + n * U) + TINY) @ np.abs(v) + U * np.abs(o)}
    with np.errstate(divide="ignore"):
        lse = np.where(row, top[:, 0] + np.log(np.where(total[:, 0] == 0, 1.0, total[:, 0])), -np.inf)
    got["lse"], got["lse_off"] = lse, worst[:, 0] + (n + 16) * U + 4 * U * np.abs(np.where(row, lse, 0.0)) + 4 * U * np.abs(np.where(row, top[:, 0], 0.0))
    if dout is None:
        return got
    g = np.where(row[:, None], dout.astype(np.float64), 0.0)
    gv, dot = g @ v.T, (g * o).sum(1, keepdims=True)
    slope_of = scale * (1.0 - t * t)
    ds = np.where(ok, w * (gv - dot) * slope_of, 0.0)
    got["dq"], got["dk"], got["dv"] = ds @ k, ds.T @ q, w.T @ g
    # weights in the gradient come from lse, which has errors of its own
    rel = off + got["lse_off"][:, None] + 8 * U
    m = q.shape[0]
    got["dv_off"] = (w * (rel + m * U) + TINY).T @ np.abs(g)
    inner = d * U * (np.abs(g) @ np.abs(v).T) + d * U * (np.abs(g) * np.abs(o)).sum(1, keepdims=True) + (np.abs(g) * got["o_off"]).sum(1, keepdims=True)
    bend = np.zeros_like(off) if cap is None else 2 * (off / cap + 8 * U) * abs(scale)     # of 1 - t^2
    ds_off = np.where(ok, w * (np.abs(slope_of) * (inner + (rel + 8 * U) * np.abs(gv - dot)) + bend * np.abs(gv - dot)), 0.0)
    ds_off = ds_off + np.where(ok, TINY * np.abs(slope_of) * (np.abs(gv - dot) + 1), 0.0)     # (or the product with a weight)
    got["dq_off"] = (ds_off + n * U * np.abs(ds)) @ np.abs(k)
    got["dk_off"] = (ds_off + m * U * np.abs(ds)).T @ np.abs(q)
    return got


def attention(q, k, v, *, scale=None, causal=False, start=None, lengths=None, prefix=None,
              documents=None, slopes=None, cap=None, dout=None):
    """All heads: o, lse (and dq, dk, dv), each with its bound under `name + "_off"`."""
    batch, hq, lq, d = q.shape
    hkv, lk = k.shape[1:3]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    names = {"o": q.shape, "lse": q.shape[:3]}
    if dout is not None:
        names |= {"dq": q.shape, "dk": k.shape, "dv": v.shape}
    out = {n + e: np.zeros(s) for n, s in names.items() for e in ("", "_off")}

    def of(x, b):
        return None if x is None else int(x if np.ndim(x) == 0 else x[b])
    for b in range(batch):
        p, ok = pairs(lq, lk, causal=causal, start=of(start, b), length=of(lengths, b), prefix=of(prefix, b) or 0,
                      documents=None if documents is None else documents[b])
        for h in range(hq):
            kv = h // (hq // hkv)
            one = head(q[b, h], k[b, kv], v[b, kv], p, ok, scale, cap, None if slopes is None else float(slopes[h]),
                       None if dout is None else dout[b, h])
            for n in out:
                if n[:2] in ("dk", "dv"):
                    out[n][b, kv] += one[n]
                else:
                    out[n][b, h] = one[n]
    if dout is not None:           # the sum over the heads of a group
        for n in ("dk", "dv"):
            out[n + "_off"] += (hq // hkv) * U * np.abs(out[n])
    return out


def rotary_matrix(position, size, dims, frequencies, stretch=1.0, magnitude=1.0, interleaved=False):
    """The matrix that turns one row."""
    m = np.eye(size)
    for i in range(dims // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + dims // 2)
        angle = position * frequencies[i] / stretch
        c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
        m[a, a], m[a, b], m[b, a], m[b, b] = c, -s, s, c
    return m


def rotary(x, positions, *, base=10000.0, frequencies=None, dims=None, interleaved=False,
           stretch=1.0, magnitude=1.0, weight=None, eps=1e-6, dy=None):
    """y, or with dy (dx, dweight); row by row."""
    batch, heads, rows, size = x.shape
    dims = size - size % 2 if dims is None else dims
    if frequencies is None:
        frequencies = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    positions = np.broadcast_to(positions + np.arange(rows) if np.ndim(positions) == 0 else positions, (batch, rows))
    y, dw = np.zeros(x.shape), None if weight is None else np.zeros((heads, size))
    for b in range(batch):
        for l in range(rows):
            m = rotary_matrix(float(positions[b, l]), size, dims, frequencies, stretch, magnitude, interleaved)
            for h in range(heads):
                row = x[b, h, l].astype(np.float64)
                w = None if weight is None else (weight if weight.ndim == 1 else weight[h]).astype(np.float64)
                r = 1.0 if w is None else 1.0 / np.sqrt((row * row).mean() + eps)
                if dy is None:
                    y[b, h, l] = m @ (row if w is None else row * r * w)
                    continue
                g = m.T @ dy[b, h, l].astype(np.float64)
                if w is None:
                    y[b, h, l] = g
                    continue
                hat = row * r
                dw[h] += g * hat
                y[b, h, l] = r * (w * g - hat * (w * g * hat).mean())
    if dy is None:
        return y
    return y if weight is None else (y, dw if weight.ndim == 2 else dw.sum(0))


def sample(row, u, temperature=1.0, top_k=None, top_p=1.0, min_p=0.0):
    """The token of one row, from a list of (weight, number) sorted as a person would."""
    from fractions import Fraction
    live = [(float(x), i) for i, x in enumerate(row) if not np.isnan(x) and x != -np.inf]
    if not live:
        return -1
    live.sort(key=lambda t: (-t[0], t[1]))
    if temperature <= 0:
        return live[0][1]
    top = live[0][0]
    weights = [(1.0 if x == top else float(np.exp((x - top) / temperature)), i) for x, i in live]
    if top_k:
        weights = weights[:top_k]
    if top_p < 1.0:
        # the part of the sum is a product in float64: 0.9 of 40 equal weights is 36 of them, although the float64 0.9 is above 0.9
        goal = Fraction(top_p * float(sum(Fraction(w) for w, _ in weights)))
        run, keep = Fraction(0), []
        for w, i in weights:
            if run < goal or not keep:
                keep.append((w, i))
            run += Fraction(w)
        weights = keep
    weights = sorted((i, w) for w, i in weights if w >= min_p)
    goal = Fraction(float(u)) * sum(Fraction(w) for _, w in weights)
    run = Fraction(0)
    for i, w in weights:
        run += Fraction(w)
        if run > goal:
            return i
    return weights[-1][0]
