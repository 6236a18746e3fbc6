"""`nn.attention` on the device where many rows give blocks of eight waves, and the precision of its products."""
import numpy as np
import pytest

import delayrepay_amd as dr
from delayrepay_amd import nn
from oracle import nn_oracle
from tests import nn_precision

pytestmark = pytest.mark.gpu
NAN, INF = np.float32("nan"), np.float32("inf")


def _ranges_of_eight_waves(b, hq, hkv, lq, lk, d, causal=False, documents=None, **_):
    """Key ranges of a call whose blocks have eight waves, by the kernels' rule; None for other calls."""
    rows, heads = hq // hkv * lq, b * hkv
    if rows <= 64 or (documents is None and heads * -(-rows // 16) * lk * d <= 25000000) or heads * -(-rows // 256) < 256:
        return None
    blocks = heads * -(-rows // 256)
    want = 64 if documents is not None else 512 if causal else 256
    ranges = min(1 if blocks >= want else -(-want // blocks), -(-lk // 256))
    chunk = -(-(-(-lk // ranges)) // 64) * 64
    return -(-lk // chunk)


def _documents(batch, n):
    rs = np.random.RandomState(n)
    return np.stack([np.repeat(np.arange(n), rs.randint(1, n // 3, n))[:n] for _ in range(batch)]).astype(np.int32)


LENGTHS = np.array([290, 555], np.int32)
# size, options, key ranges: each head size's kernel, 256-row blocks with a remainder, all kinds of masks
EIGHT = [((2, 64, 32, 401, 300, 32), dict(causal=True), 2),
         ((2, 64, 32, 385, 300, 32), dict(documents=_documents(2, 300), causal=True, slopes=np.linspace(0, 0.3, 64).astype(np.float32)), 1),
         ((2, 64, 32, 401, 555, 64), dict(causal=True, lengths=LENGTHS, prefix=70), 2),
         ((2, 64, 32, 400, 555, 80), dict(causal=True, documents=_documents(2, 555), lengths=LENGTHS, cap=3.0), 1),
         ((2, 66, 33, 391, 270, 96), dict(causal=True, slopes=np.linspace(0, 0.3, 66).astype(np.float32), cap=5.0), 2),
         ((2, 64, 32, 401, 290, 128), dict(causal=True, start=-7), 2),
         ((2, 64, 32, 401, 290, 127), dict(cap=4.0, scale=0.3), 1)]


@pytest.mark.parametrize("size,how,ranges", EIGHT, ids=[str(c[0]) for c in EIGHT])
def test_blocks_of_eight_waves(size, how, ranges):
    assert _ranges_of_eight_waves(*size, **how) == ranges
    b, hq, hkv, lq, lk, d = size
    rs = np.random.RandomState(lq + lk + d)
    q, k, v = (rs.standard_normal(s).astype(np.float32) for s in ((b, hq, lq, d), (b, hkv, lk, d), (b, hkv, lk, d)))
    if "lengths" in how:
        for s, n in enumerate(LENGTHS):
            k[s, :, n:], v[s, :, n::2], v[s, :, n + 1::2] = NAN, INF, NAN
    dev = {n: dr.array(x) if isinstance(x, np.ndarray) else x for n, x in how.items()}
    o, lse = (x.get() for x in nn.attention(*[dr.array(x) for x in (q, k, v)], with_lse=True, **dev))
    # whole heads of both sequences, the last ones among them
    for s, h in ((0, 0), (0, hq // 2 + 1), (1, 7), (1, hq - 1)):
        n = int(how["lengths"][s]) if "lengths" in how else lk
        p, ok = nn_oracle.pairs(lq, lk, causal=how.get("causal", False), start=how.get("start"), length=n, prefix=how.get("prefix", 0),
                                documents=how["documents"][s] if "documents" in how else None)
        want = nn_oracle.head(q[s, h], k[s, h // (hq // hkv)], v[s, h // (hq // hkv)], p, ok, how.get("scale", d ** -0.5), how.get("cap"),
                              float(how["slopes"][h]) if "slopes" in how else None)
        for x, name in ((o[s, h], "o"), (lse[s, h], "lse")):
            fine = bool(np.all((x == want[name]) | (np.abs(x.astype(np.float64) - want[name]) <= 2 * want[name + "_off"])))
            assert fine, (name, s, h, np.nanmax(np.abs(x - want[name])))
    # and all of them against calls of single heads, whose blocks have four waves or 16 rows: sums of the same numbers in
    # another order, each within the oracle's bound of rows like these
    most = 4 * float(want["o_off"].max()) + 4 * float(np.abs(want["o"]).max()) * 2.0 ** -24 * lk
    masks = {n: x for n, x in dev.items() if n not in ("slopes", "documents", "lengths")}
    for s, kh in ((0, 3), (1, hkv - 1)):
        group = slice(kh * (hq // hkv), (kh + 1) * (hq // hkv))
        one = {**masks, **{n: dr.array(how[n][s:s + 1]) for n in ("documents", "lengths") if n in how}}
        if "slopes" in how:
            one["slopes"] = dr.array(how["slopes"][group])
        alone = nn.attention(*[dr.array(np.ascontiguousarray(x)) for x in (q[s:s + 1, group], k[s:s + 1, kh:kh + 1], v[s:s + 1, kh:kh + 1])], **one).get()
        assert float(np.abs(alone[0] - o[s, group]).max()) <= most


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("size", nn_precision.SIZES, ids=str)
def test_products_keep_the_precision_of_float32(size, packed):
    """The root mean square error on random data, which a lost part of the matrix products would raise tenfold:
    forward by the kernels of many rows (with one document) and of few, and the gradient."""
    lq, lk, d = size
    q, k, v, g = nn_precision.inputs(*size)
    want = nn_precision.attention(q, k, v, g, nn_precision.plain_product, np.float64)
    plain = {n: nn_precision.error(x, want[n]) for n, x in nn_precision.attention(q, k, v, g, nn_precision.plain_product).items()}
    dev = [dr.array(x[None, None]) for x in (q, k, v, g)]
    how = dict(documents=dr.array(np.zeros((1, lk), np.int32)), start=0) if packed and lq <= lk else {}
    o, lse = nn.attention(*dev[:3], with_lse=True, **how)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *nn.attention_grad(dev[3], *dev[:3], o, lse, **how))))
    for n, x in got.items():
        off = nn_precision.error(x.get()[0, 0], want[n])
        assert off <= nn_precision.WORST * plain[n], (n, off, plain[n])
