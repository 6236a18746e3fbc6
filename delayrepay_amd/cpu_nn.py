"""The operators of `nn` under `DELAY_CPU`: the formulas in NumPy, in 64 bits and rounded once at the end."""
import numpy as np


def narrowed(x, low, high):
    return np.clip(x, low, high).astype(np.int32)


def renumbered(x):
    return x            # (compared in 64 bits here)


def _out(outs, values, dtype):
    """Results in the arrays asked for, or as new ones."""
    done = []
    for out, value in zip(outs, values):
        if out is None:
            out = value.astype(dtype, copy=False)
        else:
            out[...] = value
        done.append(out)
    return done


def _of(x, b):
    return int(x if isinstance(x, int) else x[b])


def _sequence(q, k, how, b):
    """(rows in use, positions of the rows, which pairs count) of one sequence."""
    lq, lk = q.shape[2], k.shape[2]
    n = lk if how.lengths is None else min(max(_of(how.lengths, b), 0), lk)
    start = n - lq if how.start is None else min(max(_of(how.start, b), -1 << 30), 1 << 30)
    p, j = start + np.arange(lq), np.arange(n)
    ok = np.ones((lq, n), bool)
    if how.causal:
        prefix = 0 if how.prefix is None else _of(how.prefix, b)
        ok &= (j <= p[:, None]) | (j < prefix)
    if how.documents is not None:
        docs = how.documents[b]
        inside = (p >= 0) & (p < n)
        own = docs[np.clip(p, 0, n - 1)] if n else np.zeros(lq, docs.dtype)
        ok &= inside[:, None] & (own[:, None] == docs[:n])
    return n, p, ok


def _scores(q, k, p, ok, slope, how):
    """Scores of one head, and tanh of the capped ones."""
    with np.errstate(invalid="ignore"):
        s, t = q @ k.T * how.scale, None
    s[~np.isfinite(q).all(1)] = np.nan
    s[:, ~np.isfinite(k).all(1)] = np.nan
    if how.cap is not None:
        t = np.tanh(s / how.cap)
        s = how.cap * t
    if slope is not None:
        s = s - slope * np.abs(p[:, None] - np.arange(k.shape[0]))
    return np.where(ok, s, -np.inf), t


def _weighted(w, x):
    """w @ x in which a weight of zero takes nothing, whatever x holds."""
    fine = np.isfinite(x)
    if fine.all():
        return w @ x
    with np.errstate(invalid="ignore"):
        y = w @ np.where(fine, x, 0.0)
        for j in np.flatnonzero(~fine.all(1)):
            rows = np.flatnonzero(w[:, j])
            y[rows] += w[rows, j, None] * np.where(fine[j], 0.0, x[j])
    return y


def attention(q, k, v, how, outs):
    batch, hq, lq, size = q.shape
    group = hq // k.shape[1]
    o, lse = np.zeros(q.shape), np.full(q.shape[:3], -np.inf)
    for b in range(batch):
        n, p, ok = _sequence(q, k, how, b)
        for h in range(hq if n else 0):
            kk, vv = (x[b, h // group, :n].astype(np.float64) for x in (k, v))
            slope = None if how.slopes is None else float(how.slopes[h])
            s, _ = _scores(q[b, h].astype(np.float64), kk, p, ok, slope, how)
            top = s.max(1, keepdims=True)
            e = np.exp(s - np.where(top == -np.inf, 0.0, top))
            total = e.sum(1, keepdims=True)
            o[b, h] = _weighted(e / np.where(total == 0, 1.0, total), vv)
            with np.errstate(divide="ignore"):
                lse[b, h] = (top + np.log(total))[:, 0]
    return _out(outs, [o, lse][:len(outs)], np.float32)


def attention_grad(dout, q, k, v, o, lse, how, outs):
    batch, hq, lq, size = q.shape
    group = hq // k.shape[1]
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for b in range(batch):
        n, p, ok = _sequence(q, k, how, b)
        for h in range(hq if n else 0):
            kk, vv = (x[b, h // group, :n].astype(np.float64) for x in (k, v))
            slope = None if how.slopes is None else float(how.slopes[h])
            row = np.isfinite(lse[b, h])[:, None] | np.isnan(lse[b, h])[:, None]
            qq, g = (np.where(row, x[b, h], 0.0).astype(np.float64) for x in (q, dout))
            s, t = _scores(qq, kk, p, ok & row, slope, how)
            w = np.where(ok & row, np.exp(s - np.where(row, lse[b, h][:, None], 0.0)), 0.0)      # (a row's lse may be NaN)
            with np.errstate(invalid="ignore"):
                d = g @ vv.T - (g * np.where(row, o[b, h], 0.0)).sum(1, keepdims=True)
                ds = np.where(ok & row, w * d * (how.scale if t is None else how.scale * (1.0 - t * t)), 0.0)
            dq[b, h] = _weighted(ds, kk)
            dk[b, h // group, :n] += _weighted(ds.T, qq)
            dv[b, h // group, :n] += _weighted(w.T, g)
    return _out(outs, [dq, dk, dv], np.float32)


def _angles(shape, how):
    batch, heads, rows, size = shape
    if how.positions is None:
        p = how.first + np.arange(rows, dtype=np.float64)[None]
    else:
        p = np.asarray(how.positions, np.float64).reshape(-1, rows)
    f = how.frequencies
    if f is None:
        f = how.base ** (-2.0 * np.arange(how.dims // 2) / max(how.dims, 1))
    a = p[:, None, :, None] * (f / how.stretch)
    return how.magnitude * np.cos(a), how.magnitude * np.sin(a)


def _turn(x, c, s, how):
    y, half = x.copy(), how.dims // 2
    one, two = (slice(0, how.dims, 2), slice(1, how.dims, 2)) if how.interleaved else (slice(0, half), slice(half, how.dims))
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    return y


def _per_row(w):
    return w[:, None, :] if w.ndim == 2 else w


def rotary(x, how, outs):
    c, s = _angles(x.shape, how)
    y = x.astype(np.float64)
    if how.weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + how.eps) * _per_row(how.weight)
    return _out(outs, [_turn(y, c, s, how)], x.dtype)


def rotary_grad(dy, x, how, outs):
    c, s = _angles(dy.shape, how)
    g = _turn(dy.astype(np.float64), c, -s, how)
    if x is None:
        return _out(outs, [g], dy.dtype)
    y = x.astype(np.float64)
    r = 1.0 / np.sqrt((y * y).mean(-1, keepdims=True) + how.eps)
    hat, w = y * r, _per_row(how.weight)
    dw = (g * hat).sum((0, 2) if how.weight.ndim == 2 else (0, 1, 2))
    return _out(outs, [r * (g * w - hat * (g * w * hat).mean(-1, keepdims=True)), dw], dy.dtype)


def sample(logits, uniforms, temperature, top_k, top_p, min_p, outs):
    batch, vocabulary = logits.shape
    tokens = np.full(batch, -1, np.int64)
    for b in range(batch):
        t, k, p, m, u = (x if isinstance(x, (int, float)) else x[b].item() for x in (temperature, top_k, top_p, min_p, uniforms))
        t, p, m, u = (0.0 if x != x else min(x, 3.4028234663852886e38) for x in (t, p, m, u))
        row = np.where(np.isnan(logits[b]), -np.inf, logits[b].astype(np.float64))
        order = np.argsort(-row, kind="stable")
        top = row[order[0]]
        if top == -np.inf:
            continue
        if not t > 0.0:
            tokens[b] = order[0]
            continue
        with np.errstate(invalid="ignore"):
            w = np.where(row == top, 1.0, np.exp((row - top) * (1.0 / t)))[order]
        if 0 < k < vocabulary:
            w[k:] = 0.0
        if p < 1.0:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            keep = before < p * w.sum()
            keep[0] = True
            w[~keep] = 0.0
        w[w < min(max(m, 0.0), 1.0)] = 0.0
        by_number = np.zeros(vocabulary)
        by_number[order] = w
        run = np.cumsum(by_number)
        hit = np.flatnonzero((run > u * run[-1]) & (by_number > 0))
        tokens[b] = hit[0] if len(hit) else np.flatnonzero(by_number)[-1]
    return _out(outs, [tokens], np.int64)
