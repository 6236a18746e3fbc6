"""`nn` on the device against the oracle in float64.  Attention's tolerances are the oracle's first-order
bounds of float32 arithmetic (one each for every element), taken times two for second-order terms and
the hardware's exp2, log2 and reciprocal (an ulp each)."""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import delayrepay_amd as dr
from delayrepay_amd import hip, nn
from delayrepay_amd.devarray import ndarray
from oracle import nn_oracle

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAN, INF = np.float32("nan"), np.float32("inf")


def _put(x):
    return dr.array(x) if isinstance(x, np.ndarray) else x


def _on_device(how):
    return {k: _put(v) for k, v in how.items()}


def _near(got, want, off, what):
    got = got.get() if not isinstance(got, np.ndarray) else got
    assert got.dtype == np.float32 and got.shape == want.shape, what
    same = (got == want) | (np.isnan(got) & np.isnan(want))       # (lse of rows without keys: -inf)
    with np.errstate(invalid="ignore"):
        far = np.abs(got.astype(np.float64) - want)
    bad = ~(same | (far <= 2 * off))
    assert not bad.any(), (what, np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], off[bad][:5])


def _check(q, k, v, g=None, **how):
    """Forward (and gradient, with g) against the oracle; the operands are host arrays or (device, host) pairs."""
    host = [x[1] if isinstance(x, tuple) else x for x in (q, k, v, g)]
    dev = [x[0] if isinstance(x, tuple) else None if x is None else _put(x) for x in (q, k, v, g)]
    want = nn_oracle.attention(*host[:3], dout=host[3], **how)
    args = _on_device(how)
    o, lse = nn.attention(*dev[:3], with_lse=True, **args)
    _near(o, want["o"], want["o_off"], "o")
    _near(lse, want["lse"], want["lse_off"], "lse")
    if g is not None:
        for name, got in zip(("dq", "dk", "dv"), nn.attention_grad(dev[3], *dev[:3], o, lse, **args)):
            _near(got, want[name], want[name + "_off"], name)
    return o, lse


def _normal(seed, *shapes):
    rs = np.random.RandomState(seed)
    return [rs.standard_normal(s).astype(np.float32) for s in shapes]


def _documents(batch, n, seed):
    rs = np.random.RandomState(seed)
    return np.stack([np.repeat(np.arange(n), rs.randint(1, max(2, n // 3), n))[:n] for _ in range(batch)]).astype(np.int32)


MASKS = ["none", "causal", "prefix", "documents", "lengths", "everything"]


def _mask(name, batch, hq, lq, lk):
    rs = np.random.RandomState(lq * 1000 + lk)
    return {"none": dict(), "causal": dict(causal=True), "prefix": dict(causal=True, prefix=rs.randint(0, lk + 1, batch).astype(np.int32)),
            "documents": dict(causal=True, documents=_documents(batch, lk, lk)),
            "lengths": dict(lengths=rs.randint(0, lk + 1, batch).astype(np.int32)),
            "everything": dict(causal=True, lengths=rs.randint(0, lk + 1, batch).astype(np.int32), documents=_documents(batch, lk, lk + 1), cap=4.0,
                               start=rs.randint(-2, lk, batch).astype(np.int32), prefix=lk // 3, slopes=rs.rand(hq).astype(np.float32), scale=0.5)}[name]


# batch, query heads, key heads, rows, key rows, head size: around the kernels' tiles of 16, 32, 64 and 128
SIZES = [(1, 1, 1, 1, 1, 1), (2, 2, 1, 3, 5, 8), (1, 4, 4, 16, 33, 32), (2, 6, 2, 31, 31, 33), (1, 3, 1, 64, 63, 64), (1, 2, 2, 129, 128, 80),
         (1, 8, 2, 1, 257, 128), (2, 5, 1, 7, 65, 96), (1, 2, 1, 200, 321, 128), (3, 16, 1, 2, 130, 72), (1, 33, 1, 1, 40, 48), (1, 1, 1, 300, 40, 127)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_attention_and_its_gradient(size, mask):
    b, hq, hkv, lq, lk, d = size
    q, g, k, v = _normal(lq + lk, (b, hq, lq, d), (b, hq, lq, d), (b, hkv, lk, d), (b, hkv, lk, d))
    _check(q, k, v, g, **_mask(mask, b, hq, lq, lk))


@pytest.mark.parametrize("lq,lk", [(0, 4), (3, 0), (0, 0)])
def test_no_rows_or_no_keys(lq, lk):
    q, g, k, v = _normal(0, (2, 2, lq, 16), (2, 2, lq, 16), (2, 1, lk, 16), (2, 1, lk, 16))
    _check(q, k, v, g)
    _check(q, k, v, g, causal=True, lengths=0)


@pytest.mark.parametrize("lq", [1, 40])
def test_rows_and_sequences_without_keys(lq):
    """Their operands hold what is not finite; they give zeros, -inf and zero gradients."""
    q, g, k, v = _normal(3, (3, 4, lq, 64), (3, 4, lq, 64), (3, 2, 50, 64), (3, 2, 50, 64))
    q[0], g[0], k[1], v[1] = NAN, INF, NAN, -INF
    lengths = np.array([0, 0, 50], np.int32)
    o, lse = _check(q, k, v, g, lengths=lengths, causal=True)
    assert not o.get()[:2].any() and np.all(lse.get()[:2] == -np.inf)
    # the first rows of a causal block stand before the first key
    q[:], g[:] = _normal(4, q.shape, g.shape)
    k[1], v[1] = _normal(5, k[1].shape, v[1].shape)
    q[:, :, :lq // 2], g[:, :, :lq // 2] = NAN, NAN
    _check(q, k, v, g, causal=True, start=-(lq // 2))


@pytest.mark.parametrize("few", [True, False])
def test_keys_that_do_not_count_may_hold_anything(few):
    """Behind the length; later than the row; of another document: non-finite keys and values next to
    keys that count, in one tile with them, leave every row that does not see them alone."""
    b, hq, hkv, lk, d = 2, 4, 2, 100, 80
    lq = 3 if few else 90
    q, g, k, v = _normal(6, (b, hq, lq, d), (b, hq, lq, d), (b, hkv, lk, d), (b, hkv, lk, d))
    lengths = np.array([60, 97], np.int32)
    k[0, :, 60:], v[0, :, 60:] = INF, NAN
    k[1, :, 97:, 5], v[1, :, 97:, 70] = NAN, INF
    _check(q, k, v, g, lengths=lengths, causal=True, start=0)
    _check(q, k, v, g, lengths=lengths)
    # one key seen by the last row alone: the others keep their values
    clean = nn_oracle.attention(q, k, v, causal=True, lengths=lengths)
    k[1, 1, 96], v[1, 1, 96, 3] = NAN, -INF
    o = nn.attention(*[_put(x) for x in (q, k, v)], causal=True, lengths=_put(lengths)).get()
    off = clean["o_off"].copy()
    off[1, 2:, -1] = INF                     # (heads 2 and 3 share key head 1)
    assert np.isnan(o[1, 2:, -1]).all()
    _near(np.where(np.isfinite(off), o, 0), np.where(np.isfinite(off), clean["o"], 0), np.where(np.isfinite(off), off, 0), "o")
    # a value that is not finite where only its own column meets it
    k[1, 1, 96] = 0.5
    o = nn.attention(*[_put(x) for x in (q, k, v)], causal=True, lengths=_put(lengths)).get()
    assert np.all(o[1, 2:, -1, 3] == -np.inf) and np.isfinite(np.delete(o[1, 2:, -1], 3, axis=-1)).all() and np.isfinite(o[1, 2:, :-1]).all()
    # the gradient: rows that do not see the key
    dev = [_put(x) for x in (q, k, v)]
    o, lse = nn.attention(*dev, causal=True, lengths=_put(lengths), with_lse=True)
    dq = nn.attention_grad(_put(g), *dev, o, lse, causal=True, lengths=_put(lengths))[0].get()
    assert np.isfinite(dq[1, 2:, :-1]).all() and np.isfinite(dq[:, :2]).all() and np.isnan(dq[1, 2:, -1]).any()


def test_rows_that_do_not_see_a_key_leave_its_gradient_alone():
    q, g, k, v = _normal(7, (1, 2, 70, 64), (1, 2, 70, 64), (1, 1, 70, 64), (1, 1, 70, 64))
    want = nn_oracle.attention(q[:, :, :10], k, v, dout=g[:, :, :10], causal=True, start=0)
    q[0, 1, 10], g[0, 0, 10, 3] = NAN, INF
    dev = [_put(x) for x in (q, k, v)]
    o, lse = nn.attention(*dev, causal=True, with_lse=True)
    _, dk, dv = (x.get() for x in nn.attention_grad(_put(g), *dev, o, lse, causal=True))
    assert np.isnan(dk[0, 0, :11]).any() and np.isfinite(dk[0, 0, 11:]).all() and np.isfinite(dv[0, 0, 11:]).all()
    assert np.all(dv[0, 0, :11, 3] == INF) | np.isnan(dv[0, 0, :11, 3]).all() and want["dk"].any()


@pytest.mark.parametrize("lq", [2, 140])
def test_strides_and_alignment(lq):
    """Heads behind rows in memory, rows that are not 16-byte aligned, a last axis that is not dense,
    operands stretched over the batch, results in views."""
    b, hq, hkv, lk, d = 2, 4, 2, 150, 64
    rs = np.random.RandomState(8)
    want = None
    for kind in ("heads last", "odd", "backwards", "not dense"):
        def make(h, n):
            if kind == "heads last":
                x = rs.standard_normal((b, n, h, d)).astype(np.float32)
                return dr.array(x).transpose((0, 2, 1, 3)), x.transpose(0, 2, 1, 3)
            if kind == "odd":
                x = rs.standard_normal((b, h, n, d + 3)).astype(np.float32)
                return dr.array(x)[..., 1:d + 1], x[..., 1:d + 1]
            if kind == "backwards":
                x = rs.standard_normal((b, h, n, d)).astype(np.float32)
                return dr.array(x)[:, ::-1, ::-1], x[:, ::-1, ::-1]
            x = rs.standard_normal((b, h, d, n)).astype(np.float32)
            return dr.array(x).transpose((0, 1, 3, 2)), x.transpose(0, 1, 3, 2)
        q, g, k, v = make(hq, lq), make(hq, lq), make(hkv, lk), make(hkv, lk)
        _check(q, k, v, g, causal=True, documents=_documents(b, lk, 3))
    # one key and value for the whole batch
    q, g, k, v = _normal(9, (3, 4, lq, 48), (3, 4, lq, 48), (1, 2, 77, 48), (1, 2, 77, 48))
    wide = [dr.broadcast_to(dr.array(x), (3, 2, 77, 48)) for x in (k, v)]
    full = [np.broadcast_to(x, (3, 2, 77, 48)) for x in (k, v)]
    _check(q, (wide[0], full[0]), (wide[1], full[1]), g, causal=True)
    # results in views of larger arrays; the rest of these stays
    want = nn_oracle.attention(q, *full, dout=g, causal=True)
    big = [dr.array(np.full((3, n, h, 50), 7, np.float32)) for n, h in ((lq, 4), (lq, 4), (77, 2), (77, 2))]
    views = [x[..., 1:49].transpose((0, 2, 1, 3)) for x in big]
    lse = dr.array(np.zeros((3, 4, lq), np.float32))
    dev = [dr.array(q), *wide]
    got = nn.attention(*dev, causal=True, with_lse=True, out=(views[0], lse))
    assert got[0] is views[0] and got[1] is lse
    nn.attention_grad(dr.array(g), *dev, views[0], lse, causal=True, out=views[1:])
    for x, y, name in zip(big, views, ("o", "dq", "dk", "dv")):
        _near(y, want[name], want[name + "_off"], name)
        assert np.all(x.get()[..., :1] == 7) and np.all(x.get()[..., 49:] == 7)


# the same for calls that are not small: more than 64 rows of a key head, and many of them in all
LARGE = [(2, 16, 8, 80, 1301, 128), (2, 16, 8, 80, 2100, 81), (2, 16, 8, 80, 5000, 33), (1, 30, 10, 131, 3100, 32)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("size", LARGE, ids=str)
def test_attention_and_its_gradient_of_many_rows(size, mask):
    b, hq, hkv, lq, lk, d = size
    q, g, k, v = _normal(lq + lk, (b, hq, lq, d), (b, hq, lq, d), (b, hkv, lk, d), (b, hkv, lk, d))
    _check(q, k, v, g, **_mask(mask, b, hq, lq, lk))


def test_many_rows_and_keys_that_do_not_count():
    """Behind the length, later than the row, in rows without keys: what is not finite stays where it is."""
    b, hq, hkv, lq, lk, d = 2, 16, 8, 80, 1300, 128
    q, g, k, v = _normal(23, (b, hq, lq, d), (b, hq, lq, d), (b, hkv, lk, d), (b, hkv, lk, d))
    lengths = np.array([1250, 0], np.int32)
    k[0, :, 1250:], v[0, :, 1250:] = INF, NAN
    k[1], v[1], q[1], g[1] = NAN, -INF, INF, NAN
    o, lse = _check(q, k, v, g, lengths=lengths, causal=True)
    assert not o.get()[1].any() and np.all(lse.get()[1] == -np.inf)
    clean = nn_oracle.attention(q, k, v, causal=True, lengths=lengths)
    # a key that the last row alone sees, and a value that is infinite in one column
    k[0, 1, 1249] = NAN
    v[0, 2, 1249, 70] = -INF
    dev = [_put(x) for x in (q, k, v)]
    o, lse = nn.attention(*dev, causal=True, lengths=_put(lengths), with_lse=True)
    got = o.get()
    assert np.isnan(got[0, 2:4, -1]).all() and np.all(got[0, 4:6, -1, 70] == -INF)
    keep = np.ones(got.shape, bool)
    keep[0, 2:4, -1] = False
    keep[0, 4:6, -1, 70] = False
    _near(np.where(keep, got, 0), np.where(keep, clean["o"], 0), np.where(keep, clean["o_off"], 0), "o")
    dq, dk, dv = (x.get() for x in nn.attention_grad(_put(g), *dev, o, lse, causal=True, lengths=_put(lengths)))
    assert np.isfinite(dq[0, :, :-1]).all() and not dq[1].any() and not dk[1].any() and not dv[1].any()
    assert np.isnan(dq[0, 2:4, -1]).any() and np.isfinite(dk[0, 3:]).all() and np.isfinite(dv[0, 3:]).all()


def test_options_that_follow_each_other():
    """What is remembered of a call's geometry is told apart by every option of it."""
    q, k, v, g = _normal(21, (2, 2, 5, 16), (2, 2, 9, 16), (2, 2, 9, 16), (2, 2, 5, 16))
    for how in (dict(), dict(start=1), dict(start=0), dict(start=np.array([1, 3], np.int32)), dict(prefix=1), dict(prefix=0), dict(prefix=np.array([7, 6], np.int32)),
                dict(cap=1.0), dict(scale=1.0), dict(start=1), dict()):
        _check(q, k, v, g, causal=True, **how)


def test_results_over_operands():
    q, k, v = _normal(10, (2, 4, 150, 32), (2, 4, 150, 32), (2, 4, 150, 32))
    want = nn_oracle.attention(q, k, v, causal=True)
    for i in range(3):
        dev = [_put(x) for x in (q, k, v)]
        nn.attention(*dev, causal=True, out=dev[i])
        _near(dev[i], want["o"], want["o_off"], i)
    dev = [_put(x) for x in (q, k, v)]
    column = dr.array(np.zeros((2, 4, 32, 150), np.float32)).transpose((0, 1, 3, 2))
    nn.attention(*dev, causal=True, out=column)
    _near(column, want["o"], want["o_off"], "a result that is not dense")


def test_long_axis_joined_from_many_blocks():
    """One row against 70000 keys and 200 rows against 5000: the ranges' results are joined."""
    q, k, v = _normal(11, (1, 8, 1, 128), (1, 2, 70000, 128), (1, 2, 70000, 128))
    k[0, 0, 60000] = q[0, 1, 0] * 3          # one key that outweighs the others, far into the axis
    _check(q, k, v, lengths=np.array([69999], np.int32), causal=True)
    q, k, v = _normal(12, (1, 2, 200, 64), (1, 1, 5000, 64), (1, 1, 5000, 64))
    _check(q, k, v, causal=True, cap=5.0)
    q, k, v = _normal(13, (1, 32, 1, 64), (1, 1, 3000, 64), (1, 1, 3000, 64))
    _check(q, k, v, causal=True, lengths=np.array([700], np.int32))      # (most ranges hold nothing)


def test_offsets_past_32_bits():
    """A cache whose last rows lie more than 2^31 elements behind its first."""
    n, pitch, d = 70000, 32768, 32
    base = ndarray((1, 1, n, pitch), np.float32)
    view = dr.NPArray(base[..., pitch - d:])
    k, q, g = _normal(14, (1, 1, n, d), (1, 2, 1, d), (1, 2, 1, d))
    view[...] = dr.array(k)
    _check(q, (view, k), (view, k), causal=True)
    few = np.s_[:, :, n - 300:]
    _check(np.tile(q, (1, 1, 150, 1)), (view[few], k[few]), (view[few], k[few]), np.tile(g, (1, 1, 150, 1)), causal=True)


def test_scores_far_from_zero():
    """Large scores keep their statistics: weights come from differences to the largest."""
    q, k, v, g = _normal(15, (1, 2, 50, 64), (1, 2, 90, 64), (1, 2, 90, 64), (1, 2, 50, 64))
    _check(q * 30, k * 30, v, g)
    _check(q * 30, k * 30, v, g, cap=50.0)
    _check(q * 1e-3, k * 1e-3, v * 1e20, g)


def test_equal_calls_give_equal_bits():
    q, k, v, g = _normal(16, (2, 8, 300, 64), (2, 2, 300, 64), (2, 2, 300, 64), (2, 8, 300, 64))
    dev = [_put(x) for x in (q, k, v, g)]
    first = None
    for _ in range(4):
        o, lse = nn.attention(*dev[:3], causal=True, with_lse=True)
        bits = [x.get().tobytes() for x in (o, lse, *nn.attention_grad(dev[3], *dev[:3], o, lse, causal=True))]
        assert first is None or bits == first
        first = bits


# ---- rotary positions ------------------------------------------------------------------------
# A turned element is two products and their sum, its cosine and sine 2 ulp of float32: 2 |x| (2 + 2) u, and
# with a norm the mean of `size` squares, a root and a quotient: (size / 2 + 6) u more.

ROTARY = [(1, 1, 1, 2), (2, 3, 5, 8), (1, 40, 3, 128), (2, 2, 33, 80), (3, 1, 7, 33), (1, 9, 70, 256), (1, 2, 2, 512), (2, 1, 300, 64), (1, 17, 2, 96)]


def _rotary_off(x, weight, magnitude, u):
    size = np.abs(x).max(-1, keepdims=True).astype(np.float64)
    if weight is None:
        return 8 * u * magnitude * size + np.zeros(x.shape)
    r = 1.0 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-12)
    return (8 + x.shape[-1] / 2 + 6) * u * magnitude * size * r * np.abs(weight).max() + np.zeros(x.shape)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", ROTARY, ids=str)
def test_rotary_and_its_gradient(size, interleaved, dtype):
    b, h, n, d = size
    rs = np.random.RandomState(d + n)
    x, g = (rs.standard_normal(size).astype(dtype) for _ in range(2))
    u = np.finfo(dtype).eps / 2
    # in 64 bits the angle itself is rounded: position * frequency, up to 2^20, and the frequency's own power of two
    slack = 0 if dtype == np.float32 else (1 << 20) * 40 * 2.0 ** -53
    ways = [dict(), dict(dims=max(2, d // 4 * 2), stretch=3.0), dict(weight=rs.rand(d).astype(dtype)), dict(weight=rs.rand(h, d).astype(dtype), magnitude=1.25, base=50000.0),
            dict(dims=2 * (d // 4), frequencies=rs.rand(d // 4), weight=rs.rand(h, d).astype(dtype))]
    for way in ways:
        at = rs.randint(0, 1 << 20, (b, n)) if len(way) % 2 else rs.randint(-5, 1000, n).astype(np.int32)
        for positions in (at, 77):
            how = dict(way, interleaved=interleaved)
            dev = _on_device(how)
            got = nn.rotary(dr.array(x), _put(positions) if np.ndim(positions) else positions, **dev).get()
            want = nn_oracle.rotary(x, positions, **how)
            off = _rotary_off(x, way.get("weight"), way.get("magnitude", 1.0), u)
            assert got.dtype == dtype and np.all(np.abs(got - want) <= 2 * (off + slack * (1 + np.abs(want)))), (way.keys(), np.abs(got - want).max())
            got = nn.rotary_grad(dr.array(g), dr.array(x), _put(positions) if np.ndim(positions) else positions, **dev)
            want = nn_oracle.rotary(x, positions, dy=g, **how)
            if "weight" not in way:
                off = _rotary_off(g, None, way.get("magnitude", 1.0), u)
                assert np.all(np.abs(got.get() - want) <= 2 * (off + slack * (1 + np.abs(want))))
                continue
            # dx: r (w g - hat mean): the terms are at most r max|w| max|g| (1 + |hat|), hat at most sqrt(d)
            r = 1.0 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
            hat = np.abs(x * r)
            top = np.abs(g).max(-1, keepdims=True) * way.get("magnitude", 1.0) * np.abs(way["weight"]).max()
            off = (3 * d / 2 + 30) * u * r * top * (1 + hat * hat.mean(-1, keepdims=True))
            assert np.all(np.abs(got[0].get() - want[0]) <= 2 * (off + slack * r * top * (2 + hat))), (way.keys(), np.abs(got[0].get() - want[0]).max())
            # dweight: b n (or b n h) terms of g hat
            terms = (2 * top / np.abs(way["weight"]).max() * hat)
            total = terms.sum((0, 2)) if way["weight"].ndim == 2 else terms.sum((0, 1, 2))
            count = b * n * (1 if way["weight"].ndim == 2 else h)
            assert got[1].get().shape == way["weight"].shape
            assert np.all(np.abs(got[1].get() - want[1]) <= 2 * ((count + d / 2 + 20) * u * total + slack * total))


def test_rotary_in_place_views_and_empty():
    rs = np.random.RandomState(5)
    qkv = rs.standard_normal((2, 9, 7, 64)).astype(np.float32)            # rows, then 3 query, 2 key, 2 value heads
    dev = dr.array(qkv)
    w = rs.rand(5, 64).astype(np.float32)
    part = dev[:, :, :5].transpose((0, 2, 1, 3))
    nn.rotary(part, 100, weight=dr.array(w), out=part)                     # queries and keys, where they are
    want = nn_oracle.rotary(qkv[:, :, :5].transpose(0, 2, 1, 3), 100, weight=w)
    got = dev.get()
    assert np.allclose(got[:, :, :5].transpose(0, 2, 1, 3), want, rtol=0, atol=2 * (8 + 38) * 2.0 ** -24 * np.abs(want).max() * 2)
    assert np.array_equal(got[:, :, 5:], qkv[:, :, 5:])
    # shifted over itself: through a copy
    x = rs.standard_normal((1, 1, 20, 32)).astype(np.float32)
    dev = dr.array(x)
    nn.rotary(dev[:, :, :19], 0, out=dev[:, :, 1:])
    plain = nn.rotary(dr.array(x[:, :, :19]), 0).get()
    assert np.array_equal(dev.get()[:, :, 1:], plain)
    odd = dr.array(np.zeros((1, 1, 19, 35), np.float32))
    nn.rotary(dr.array(x[:, :, :19]), 0, out=odd[..., 3:])                 # rows that are not 16-byte aligned
    assert np.array_equal(odd.get()[..., 3:], plain)
    assert nn.rotary(dr.array(np.zeros((2, 0, 3, 8), np.float32)), 0).shape == (2, 0, 3, 8)
    dx, dw = nn.rotary_grad(*[dr.array(np.zeros((2, 3, 0, 8), np.float32))] * 2, 0, weight=dr.array(np.ones(8, np.float32)))
    assert dx.shape == (2, 3, 0, 8) and not dw.get().any()


def test_rotary_weights_of_no_heads_and_of_equal_heads():
    """No heads: a gradient of zeros, written over what stood there.  One row of weights broadcast to the heads: a gradient for each."""
    ones = dr.array(np.ones(8, np.float32))
    dw = dr.array(np.full(8, 7, np.float32))
    empty = dr.array(np.zeros((2, 0, 3, 8), np.float32))
    nn.rotary_grad(empty, empty, 0, weight=ones, out=(dr.array(np.zeros((2, 0, 3, 8), np.float32)), dw))
    assert not dw.get().any()
    assert nn.rotary_grad(empty, empty, 0, weight=dr.array(np.zeros((0, 8), np.float32)))[1].shape == (0, 8)
    x, g, w = _normal(22, (2, 5, 6, 64), (2, 5, 6, 64), (64,))
    dev = [dr.array(a) for a in (g, x)]
    same = dr.broadcast_to(dr.array(w)[None], (5, 64))
    each = dr.array(np.tile(w, (5, 1)))
    for a, b in zip(nn.rotary_grad(*dev, 3, weight=same), nn.rotary_grad(*dev, 3, weight=each)):
        assert a.shape == b.shape and a.get().tobytes() == b.get().tobytes()
    assert nn.rotary(dev[1], 3, weight=same).get().tobytes() == nn.rotary(dev[1], 3, weight=each).get().tobytes()


# ---- tokens ----------------------------------------------------------------------------------

def _draws(logits, u, **how):
    """Tokens against the oracle's exact ones."""
    args = {k: _put(v) for k, v in how.items()}
    got = nn.sample(dr.array(logits), dr.array(u), **args).get()
    assert got.dtype == np.int64
    for b, (row, x) in enumerate(zip(logits, u)):
        one = {k: (v[b].item() if isinstance(v, np.ndarray) else v) for k, v in how.items()}
        assert got[b] == nn_oracle.sample(row, x, **one), (b, one, x)


WAYS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(top_k=1), dict(top_k=7), dict(top_p=0.5), dict(top_p=1e-9), dict(min_p=0.3), dict(min_p=1.0),
        dict(top_k=40, top_p=0.9, min_p=0.01, temperature=1.7), dict(top_k=10 ** 6, top_p=1.0)]


@pytest.mark.parametrize("how", WAYS, ids=str)
@pytest.mark.parametrize("vocabulary", [1, 2, 63, 511, 513, 4097, 32000])
def test_sample(vocabulary, how):
    rs = np.random.RandomState(vocabulary)
    logits = (rs.standard_normal((6, vocabulary)) * 3).astype(np.float32)
    logits[4:] = np.round(logits[4:])                      # many equal logits
    _draws(logits, rs.rand(6), **how)


@pytest.mark.parametrize("how", WAYS, ids=str)
def test_sample_of_equal_and_missing_logits(how):
    rs = np.random.RandomState(1)
    n = 3000
    logits = np.zeros((8, n), np.float32)
    logits[1] = -0.0
    logits[1, ::2] = 0.0                                    # (-0 and 0 are equal)
    logits[2] = -np.inf
    logits[3, :] = -np.inf
    logits[3, 1234] = -80.0
    logits[4] = NAN
    logits[5] = rs.standard_normal(n)
    logits[5, 100:200] = NAN
    logits[6, 50], logits[6, 70] = np.inf, np.inf
    logits[7] = np.finfo(np.float32).min
    logits[7, 5:9] = np.finfo(np.float32).max
    for u in (0.0, 0.25, 0.999999999):
        _draws(logits, np.full(8, u), **how)


def test_sample_with_parameters_for_each_row():
    rs = np.random.RandomState(2)
    logits = (rs.standard_normal((40, 5000)) * 2).astype(np.float32)
    f = np.float32
    _draws(logits, rs.rand(40), temperature=rs.choice([0.0, 0.5, 1.0, 2.0], 40).astype(f), top_k=rs.choice([-1, 0, 1, 10, 4999, 5000, 6000], 40).astype(np.int32),
           top_p=rs.choice([0.1, 0.9, 1.0], 40).astype(f), min_p=rs.choice([0.0, 0.05], 40).astype(f))
    _draws(logits, rs.rand(40).astype(f), top_k=rs.randint(1, 100, 40))          # int64, float32 uniforms
    wide = (rs.standard_normal((3, 9000)) * 2).astype(f)
    got = nn.sample(dr.array(wide)[:, 3:8003], dr.array(np.array([0.1, 0.5, 0.9]))).get()       # a row pitch
    assert got.tolist() == [nn_oracle.sample(r, u) for r, u in zip(wide[:, 3:8003], (0.1, 0.5, 0.9))]
    tokens = dr.array(np.full(9, 5, np.int64))
    nn.sample(dr.array(logits[:3]), dr.array(np.array([0.1, 0.5, 0.9])), out=tokens[::3])
    assert tokens.get()[1::3].tolist() == [5, 5, 5] and tokens.get()[::3].tolist() == [nn_oracle.sample(r, u) for r, u in zip(logits, (0.1, 0.5, 0.9))]
    assert nn.sample(dr.array(np.zeros((0, 5), f)), dr.array(np.zeros(0))).shape == (0,)


@pytest.mark.parametrize("how", [dict(top_k=1), dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_k=255), dict(top_k=257), dict(top_k=3000, min_p=0.01), dict(top_p=0.95), dict()], ids=str)
@pytest.mark.parametrize("vocabulary", [65535, 70001, 131072])
def test_sample_of_long_rows(vocabulary, how):
    """Beginnings that the first part of the row says much about, little, and nothing."""
    rs = np.random.RandomState(vocabulary)
    logits = (rs.standard_normal((6, vocabulary)) * 2.5).astype(np.float32)
    logits[1] = np.sort(logits[1])                         # the largest come last
    logits[2] = np.sort(logits[2])[::-1]
    logits[3] = np.round(logits[3])                        # many equal ones
    logits[4, :20000] = NAN                                # fewer than k in the first part
    logits[5] = -np.inf
    logits[5, [5, 17000, vocabulary - 1]] = [1.0, 2.0, 2.0]
    _draws(logits, rs.rand(6), **how)


def test_sample_of_rows_in_large_parts():
    """Rows so long that their parts are no multiple of what a wave reads at a time; against running sums in 64 bits,
    whose roundings (2e6 of 2^-53) a draw meets with a probability of 1e-9."""
    rs = np.random.RandomState(6)
    n = 2200003
    logits = (rs.standard_normal((2, n)) * 2.5).astype(np.float32)
    u = np.array([0.37, 0.81])
    dev, draw = dr.array(logits), dr.array(u)
    for how in (dict(), dict(top_p=0.6), dict(top_k=200), dict(top_k=5000, top_p=0.9), dict(min_p=0.01)):
        got = nn.sample(dev, draw, **how).get()
        for row, x, token in zip(logits.astype(np.float64), u, got):
            w = np.exp(row - row.max())
            order = np.argsort(-row, kind="stable")
            w[order[how.get("top_k", n):]] = 0.0
            run = np.cumsum(w[order])
            w[order[1:][run[:-1] >= how.get("top_p", 2.0) * run[-1]]] = 0.0
            w[w < how.get("min_p", 0.0)] = 0.0
            run = np.cumsum(w)
            assert token == np.searchsorted(run, x * run[-1], side="right"), how


@pytest.mark.parametrize("vocabulary", [40, 5000])
def test_sample_with_parameters_at_their_ends(vocabulary):
    """Out of range in an array: the nearest in it.  The smallest temperatures leave the largest logits."""
    rs = np.random.RandomState(3)
    logits = np.round(rs.standard_normal((6, vocabulary)) * 2).astype(np.float32)
    u = rs.rand(6)
    f = np.float32
    _draws(logits, u, top_p=np.array([0.0, -0.5, -1e30, -2.0, 1.5, INF], f))
    _draws(logits, u, top_p=np.array([0.0, -0.5, -1e30, -2.0, 1.5, INF], f), top_k=30)
    _draws(logits, u, top_p=np.array([0.0, -0.5, -1e30, -2.0, 1.5, INF], f), top_k=min(vocabulary - 1, 3000), temperature=1e30)      # (nearly equal weights)
    for temperature in (5e-324, 1e-300, 1e-45, np.full(6, 1e-45, f), np.full(6, np.finfo(f).max)):
        _draws(logits, u, temperature=temperature)
        _draws(logits, u, temperature=temperature, top_k=5, top_p=0.5, min_p=0.9)


@pytest.mark.parametrize("how", [dict(), dict(top_p=0.9), dict(top_k=3), dict(top_k=3, top_p=0.7, min_p=0.1)], ids=str)
def test_sample_of_extreme_logits(how):
    """What is not a number or -inf is never drawn, at no temperature; next to the ends of float32."""
    rs = np.random.RandomState(4)
    info, f = np.finfo(np.float32), np.float32
    logits = np.tile(np.array([NAN, -INF, info.min, info.min, 0, NAN, -INF], f), (7, 100))
    logits[1] = np.where(logits[1] == 0, np.nextafter(info.min, f(0)), logits[1])
    logits[2] = np.where(logits[2] == 0, info.max, logits[2])
    logits[3, 300:] = INF
    logits[4, 4] = INF                                    # one, next to the largest finite ones
    logits[4, 11] = info.max
    logits[5] = np.where(logits[5] == 0, -INF, logits[5])
    logits[6] = np.where(logits[6] == 0, info.tiny, logits[6])
    for temperature in (1.0, 1e30, 1e-40, float(info.max), np.full(7, info.max), np.full(7, 1e20, f)):
        _draws(logits, rs.rand(7), temperature=temperature, **how)


def test_sample_from_the_device_generator():
    """The generator's lazy numbers are evaluated for the call; frequencies follow the weights: of 20000 draws
    each share is within five standard deviations."""
    p = np.array([0.5, 0.25, 0.125, 0.125])
    logits = dr.broadcast_to(dr.array(np.log(p).astype(np.float32)[None]), (20000, 4))
    got = np.bincount(nn.sample(logits, dr.random.device(seed=3).random(20000)).get(), minlength=4) / 20000
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / 20000))


# ---- together, recorded, and with another library ----------------------------------------------

def test_a_decoder_layer_token_by_token_agrees_with_the_whole_prompt():
    """Norm and positions, a cache written row by row, attention over it, tokens drawn: one step at a time
    as all at once."""
    rs = np.random.RandomState(6)
    batch, hq, hkv, n, d, vocabulary = 2, 4, 2, 12, 32, 100
    x = rs.standard_normal((batch, n, 48)).astype(np.float32)
    wq, wk, wv, wo = (rs.standard_normal(s).astype(np.float32) / 7 for s in ((48, hq * d), (48, hkv * d), (48, hkv * d), (hq * d, vocabulary)))
    norm = 1 + 0.1 * rs.standard_normal((hq + hkv, d)).astype(np.float32)
    u = rs.rand(batch)
    dev = [dr.array(w) for w in (wq, wk, wv, wo)]
    weight = dr.array(norm)

    def project(rows):
        t = rows.shape[1]
        flat = dr.array(rows.reshape(batch * t, 48))
        return [(flat @ w).reshape((batch, t, -1, d)).transpose((0, 2, 1, 3)) for w in dev[:3]]

    def answer(o):
        logits = o.transpose((0, 2, 1, 3)).reshape((batch * o.shape[2], hq * d)) @ dev[3]
        return logits.reshape((batch, -1, vocabulary))[:, -1]
    q, k, v = project(x)
    q, k = nn.rotary(q, 0, weight=weight[:hq]), nn.rotary(k, 0, weight=weight[hq:])
    whole = nn.attention(q, k, v, causal=True)
    cache = [dr.array(np.full((batch, hkv, 40, d), NAN, np.float32)) for _ in range(2)]
    for t in range(n):
        q1, k1, v1 = project(x[:, t:t + 1])
        cache[0][:, :, t:t + 1] = nn.rotary(k1, t, weight=weight[hq:])
        cache[1][:, :, t:t + 1] = v1
        one = nn.attention(nn.rotary(q1, t, weight=weight[:hq]), *cache, causal=True, lengths=dr.array(np.full(batch, t + 1, np.int32)))
        # both are the same sums in another order: 2 (d + 48 + n) roundings of terms of size about one
        assert np.abs(one.get()[:, :, 0] - whole.get()[:, :, t]).max() <= 2 * (d + 48 + n) * 2.0 ** -24 * 8
    logits = answer(whole)
    got = nn.sample(logits, dr.array(u), top_k=20, top_p=0.9)
    assert got.get().tolist() == [nn_oracle.sample(r, z, top_k=20, top_p=0.9) for r, z in zip(logits.get(), u)]


def test_recorded_and_captured_calls():
    """Recordings own their workspaces: two of them and eager calls in between leave each other's results alone."""
    q, k, v, g = _normal(17, (1, 4, 1, 64), (1, 2, 4000, 64), (1, 2, 4000, 64), (1, 4, 1, 64))
    q2, k2, v2, g2 = _normal(18, (1, 4, 130, 64), (1, 2, 130, 64), (1, 2, 130, 64), (1, 4, 130, 64))
    logits, w = _normal(19, (3, 999), (4, 64))
    sets = [[_put(x) for x in s] for s in ((q, k, v, g), (q2, k2, v2, g2))]
    weight, rows, u = _put(w), _put(logits), dr.array(np.array([0.2, 0.6, 0.9]))

    def work(s):
        o, lse = nn.attention(*s[:3], causal=True, with_lse=True)
        dq, dk, dv = nn.attention_grad(s[3], *s[:3], o, lse, causal=True)
        y = nn.rotary(o, 5, weight=weight)
        dx, dw = nn.rotary_grad(s[3], o, 5, weight=weight)
        return [o, lse, dq, dk, dv, y, dx, dw, nn.sample(rows, u, top_p=0.8)]
    plans = []
    for s in sets:
        with hip.record() as plan:
            results = work(s)
        plans.append((plan.as_graph(), results, [x.get() for x in results]))
    rs = np.random.RandomState(0)
    for turn in range(3):
        for s, (plan, results, _) in zip(sets, plans):
            for x in s:
                x[...] = dr.array(rs.standard_normal(x.shape).astype(np.float32))
            plan()
        eager = [work(s) for s in sets]
        dr.synchronize()
        for (plan, results, _), want in zip(plans, eager):
            for a, b in zip(results, want):
                assert a.get().tobytes() == b.get().tobytes(), turn
        plans[1][0]()
        plans[0][0]()
        for (plan, results, _), want in zip(plans, eager):
            for a, b in zip(results, want):
                assert a.get().tobytes() == b.get().tobytes(), turn


def test_results_follow_writes():
    """What was computed from a result or an output is computed again when it changes."""
    q, k, v = _normal(20, (1, 2, 40, 32), (1, 2, 40, 32), (1, 2, 40, 32))
    dq, dk, dv = (_put(x) for x in (q, k, v))
    out = dr.array(np.zeros((1, 2, 40, 32), np.float32))
    twice = out * 2.0
    assert not twice.get().any()
    nn.attention(dq, dk, dv, out=out)
    assert np.array_equal(twice.get(), 2 * out.get()) and out.get().any()
    lazy = dq * 2.0                       # an expression as an operand
    want = nn_oracle.attention(q * 2, k, v)
    _near(nn.attention(lazy, dk, dv), want["o"], want["o_off"], "lazy")
    dq[...] = 0.0
    want = nn_oracle.attention(q * 0, k, v)
    _near(nn.attention(lazy, dk, dv), want["o"], want["o_off"], "after a write")


def test_arrays_of_another_library():
    """A torch program's tensors without a copy: on a stream of their own, not dense, written through, outliving
    their names, and refused where they do not fit (in a child process, which imports torch first)."""
    script = textwrap.dedent("""
        import gc
        import torch
        side = torch.cuda.Stream()
        import numpy as np
        import delayrepay_amd as dr
        from delayrepay_amd import nn
        from delayrepay_amd.devarray import _LEAVING
        # made on another stream, behind long work there: the import waits for it
        big = torch.randn(4096, 4096, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                big = big @ big * 1e-4
            t = torch.full((3, 5, 7), 2.0, device="cuda")
            t += big[0, 0] * 0 + 1
            a = dr.from_dlpack(t)
        assert np.array_equal((a * 2).get(), np.full((3, 5, 7), 6, np.float32))
        # views, types, strides
        for dtype in (torch.float32, torch.float64, torch.int32, torch.int64, torch.uint8, torch.bool):
            x = (torch.arange(60, device="cuda") % 7).to(dtype).view(3, 4, 5)
            for y in (x, x.transpose(0, 2), x[:, 1:, ::2], x[1], x[:0], x[2, 3, 4]):
                assert np.array_equal(dr.from_dlpack(y).get(), y.cpu().numpy()), (dtype, y.shape)
        # writes go through, also those that read what they overwrite
        x = torch.arange(10.0, device="cuda")
        a = dr.from_dlpack(x)
        a[1:] = a[:-1] + 0.5
        dr.synchronize()
        assert x.tolist() == [0.0] + [i + 0.5 for i in range(9)], x
        a[1:] = a[:-1] * 2.0
        dr.synchronize()
        assert x.tolist() == [0.0, 0.0] + [2 * (i + 0.5) for i in range(8)], x
        # results straight into a tensor
        q, k, v = (torch.randn(2, 50, 4, 64, device="cuda").transpose(1, 2) for _ in range(3))
        o = torch.empty_like(q)
        nn.attention(*[dr.from_dlpack(y) for y in (q, k, v)], causal=True, out=dr.from_dlpack(o))
        dr.synchronize()
        s = (q @ k.transpose(2, 3) / 8).masked_fill(torch.ones(50, 50, device="cuda", dtype=torch.bool).triu(1), -1e30)
        assert (o - torch.softmax(s, -1) @ v).abs().max() < 1e-5
        # memory goes back only after the work queued here
        for _ in range(50):
            y = torch.ones(1 << 20, device="cuda")
            a = dr.from_dlpack(y)
            b = (a + 1.0)
            b.run()
            del y, a
            junk = torch.full((1 << 20,), 5.0, device="cuda")
            assert float(b.get().max()) == 2.0
            del b
        gc.collect()
        dr.synchronize()
        assert not _LEAVING or len(_LEAVING) < 20
        for bad, kind in ((torch.zeros(3, device="cuda", dtype=torch.float16), TypeError), (torch.zeros(3, device="cuda", dtype=torch.complex64), TypeError)):
            try:
                dr.from_dlpack(bad)
            except kind:
                pass
            else:
                raise AssertionError(bad.dtype)
        assert np.array_equal(dr.from_dlpack(torch.arange(3)).get(), [0, 1, 2])
        print("done")
    """)
    r = subprocess.run([sys.executable, "-u", "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout[-1500:] + r.stderr[-3000:]
