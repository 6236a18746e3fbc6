"""`nn` on the device at the ends of its arguments' ranges: numbers of 64 bits, large caches, operands next to
float32's largest or not finite, arrays of another library.  Against the oracle in float64 with its first-order bounds
(times two, as in the other tests of `nn`), or bit by bit against a call that says the same in other arguments."""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

import delayrepay_amd as dr
from delayrepay_amd import nn
from oracle import nn_oracle

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAN, INF = np.float32("nan"), np.float32("inf")


def _normal(seed, *shapes):
    rs = np.random.RandomState(seed)
    return [rs.standard_normal(s).astype(np.float32) for s in shapes]


def _all(q, k, v, g, **how):
    """o, lse, dq, dk, dv of device calls on host arrays."""
    how = {n: dr.array(x) if isinstance(x, np.ndarray) else x for n, x in how.items()}
    dev = [dr.array(x) for x in (q, k, v, g)]
    o, lse = nn.attention(*dev[:3], with_lse=True, **how)
    return [x.get() for x in (o, lse, *nn.attention_grad(dev[3], *dev[:3], o, lse, **how))]


def _same_bits(got, want):
    differ = [n for n, x, y in zip(("o", "lse", "dq", "dk", "dv"), got, want) if x.tobytes() != y.tobytes()]
    assert not differ, differ


@pytest.mark.parametrize("lq", [3, 130])
def test_numbers_of_64_bits_are_clamped(lq):
    q, g, k, v = _normal(lq, (4, 2, lq, 32), (4, 2, lq, 32), (4, 1, 150, 32), (4, 1, 150, 32))
    wide = np.array([2 ** 63 - 1, 2 ** 32 + 3, -2 ** 63, -2 ** 32 + 3])
    narrow = {"lengths": [150, 150, 0, 0], "prefix": [150, 150, 0, 0], "start": [2 ** 30, 2 ** 30, -2 ** 30, -2 ** 30]}
    for name, same in narrow.items():
        _same_bits(_all(q, k, v, g, causal=True, **{name: wide}), _all(q, k, v, g, causal=True, **{name: np.array(same, np.int32)}))
    strided = dr.array(np.stack([wide, wide * 0], 1).reshape(-1))[::2]
    dev = [dr.array(x) for x in (q, k, v)]
    want = nn.attention(*dev, lengths=dr.array(np.array(narrow["lengths"], np.int32))).get()
    _same_bits([nn.attention(*dev, lengths=strided).get()], [want])
    rs = np.random.RandomState(0)
    logits, u = dr.array(rs.standard_normal((4, 500)).astype(np.float32)), dr.array(rs.rand(4))
    assert nn.sample(logits, u, top_k=dr.array(wide)).get().tolist() == nn.sample(logits, u).get().tolist()

@pytest.mark.parametrize("size", [(2, 3, 90), (2, 40, 90), (1, 90, 700), (1, 2, 5000)], ids=str)
def test_documents_of_64_bits(size):
    """Numbers that agree in their low 32 bits, or in the high ones, are different documents."""
    b, lq, lk = size
    rs = np.random.RandomState(lk)
    names = np.array([1, 1 + (1 << 32), 1 - (1 << 32), -1, 0, 2 ** 63 - 1, -2 ** 63, 1 << 32, 7, 8])
    order = np.repeat(rs.randint(0, len(names), lk), rs.randint(1, max(2, lk // 9), lk))[:b * lk].reshape(b, lk)      # (they come back)
    q, g, k, v = _normal(lk, (b, 4, lq, 32), (b, 4, lq, 32), (b, 2, lk, 32), (b, 2, lk, 32))
    for how in (dict(), dict(causal=True, lengths=rs.randint(lk // 2, lk + 1, b).astype(np.int32))):
        _same_bits(_all(q, k, v, g, documents=names[order], **how), _all(q, k, v, g, documents=order.astype(np.int32), **how))
    dev = [dr.array(x) for x in (q, k, v)]
    wide = dr.array(np.stack([names[order], names[order] * 0], 2))[:, :, 0]              # every other number
    want = nn.attention(*dev, documents=dr.array(order.astype(np.int32))).get()
    _same_bits([nn.attention(*dev, documents=wide).get()], [want])


def test_documents_of_64_bits_all_alike_and_all_apart():
    rs = np.random.RandomState(3)
    lk = 3000
    q, g, k, v = _normal(lk, (2, 2, 70, 16), (2, 2, 70, 16), (2, 1, lk, 16), (2, 1, lk, 16))
    apart = rs.permutation(lk).astype(np.int64) << 40
    ids = np.stack([np.full(lk, -5 << 33), apart])
    _same_bits(_all(q, k, v, g, documents=ids), _all(q, k, v, g, documents=np.stack([np.zeros(lk), apart >> 40]).astype(np.int32)))


def test_recorded_documents_of_64_bits():
    """A recording and its graph renumber what the array holds when they are replayed."""
    from delayrepay_amd import hip
    rs = np.random.RandomState(4)
    q, k, v = (dr.array(x) for x in _normal(4, (2, 2, 5, 32), (2, 2, 60, 32), (2, 2, 60, 32)))
    ids = dr.array(np.zeros((2, 60), np.int64))
    with hip.record() as plan:
        out = nn.attention(q, k, v, documents=ids)
    plan.as_graph()
    for turn in range(4):
        now = rs.randint(0, 3, (2, 60)) * (1 << 32)
        ids[...] = dr.array(now)
        plan()
        want = nn.attention(q, k, v, documents=dr.array((now >> 32).astype(np.int32))).get()
        _same_bits([out.get()], [want])


def test_recorded_lengths_of_64_bits_and_gradients_of_a_part():
    """What a replay clamps and clears is what the arrays hold then."""
    from delayrepay_amd import hip
    q, g, k, v = (dr.array(x) for x in _normal(14, (2, 2, 40, 32), (2, 2, 40, 32), (2, 2, 60, 32), (2, 2, 60, 32)))
    lengths = dr.array(np.array([60, 60]))
    grads = [dr.array(np.full(x.shape, 7, np.float32)) for x in (q, k, v)]
    with hip.record() as plan:
        o, lse = nn.attention(q, k, v, lengths=lengths, with_lse=True)
        part = nn.attention(q, k, v, lengths=50, with_lse=True)
        nn.attention_grad(g, q, k, v, *part, lengths=50, out=grads)
    plan.as_graph()
    want = [x.get() for x in nn.attention_grad(g, q, k, v, *part, lengths=50)]
    for now in ([2 ** 40, 3], [0, -(2 ** 50)], [17, 2 ** 31]):
        lengths[...] = dr.array(np.array(now))
        for x in grads:
            x[...] = 7.0
        plan()
        small = dr.array(np.clip(now, 0, 60).astype(np.int32))
        _same_bits([x.get() for x in (o, lse)], [x.get() for x in nn.attention(q, k, v, lengths=small, with_lse=True)])
        _same_bits([x.get() for x in grads], want)
        assert not want[1][:, :, 50:].any()


def test_nothing_at_all_in_64_bits():
    """No sequences, no keys, no rows: results of their shapes."""
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k = (dr.array(np.ones((b, 2, n, 8), np.float32)) for n in (lq, lk))
        how = dict(lengths=dr.array(np.zeros(b, np.int64)), documents=dr.array(np.zeros((b, lk), np.int64)), start=dr.array(np.zeros(b, np.int64)))
        o, lse = nn.attention(q, k, k, with_lse=True, **how)
        dq, dk, dv = nn.attention_grad(q, q, k, k, o, lse, **how)
        assert o.shape == dq.shape == (b, 2, lq, 8) and dk.shape == dv.shape == (b, 2, lk, 8) and lse.shape == (b, 2, lq)
        assert not any(x.get().any() for x in (o, dq, dk, dv)) and np.all(lse.get() == -INF)
    assert nn.sample(dr.array(np.zeros((0, 5), np.float32)), dr.array(np.zeros(0)), top_k=dr.array(np.zeros(0, np.int64))).shape == (0,)


def test_caches_of_many_sequences():
    """One token for each of 64 sequences of up to 65536 keys, 64 heads on 8 (17 GB if the sequences did not share their keys here)."""
    b, hq, hkv, lk, d = 64, 64, 8, 65536, 64
    q, k, v = _normal(5, (b, hq, 1, d), (1, hkv, lk, d), (1, hkv, lk, d))
    lengths = (lk - 977 * np.arange(b)).astype(np.int32)
    dev = [dr.array(q)] + [dr.broadcast_to(dr.array(x), (b, hkv, lk, d)) for x in (k, v)]
    o, lse = (x.get() for x in nn.attention(*dev, causal=True, lengths=dr.array(lengths), with_lse=True))
    for s, h in ((0, 0), (17, 63), (63, 20)):
        n = int(lengths[s])
        p = np.array([n - 1])
        want = nn_oracle.head(q[s, h], k[0, h // 8, :n], v[0, h // 8, :n], p, np.ones((1, n), bool), d ** -0.5)
        assert np.all(np.abs(o[s, h] - want["o"]) <= 2 * want["o_off"]) and np.all(np.abs(lse[s, h] - want["lse"]) <= 2 * want["lse_off"])


def _near(got, want, names):
    """Within twice the oracle's bounds.  These count relative roundings; what lies below the smallest normal number, 2^-126,
    may become zero besides: of each sum at most 6 products (the parts of a float32 one) of 200 pairs, 2^-115 in all."""
    for x, name in zip(got, names):
        off = 2 * want[name + "_off"] + 2.0 ** -115
        fine = bool(np.all((x == want[name]) | (np.abs(x.astype(np.float64) - want[name]) <= off)))
        assert fine, (name, np.abs(x - want[name]).max(), off.max())


@pytest.mark.parametrize("lq", [5, 90])
def test_operands_next_to_the_largest(lq):
    """Finite numbers above bfloat16's largest, 3.39e38, are what they are, in packed operands and others.  What meets
    them is small and has one bit, so that the products are exact."""
    big = np.float32(3.395e38)
    one = np.float32(2.0 ** -126)
    names = ("o", "lse", "dq", "dk", "dv")
    shapes = (2, 2, lq, 64), (2, 2, lq, 64), (2, 1, 130, 64), (2, 1, 130, 64)
    docs = np.zeros((2, 130), np.int32)
    # (a cap: without one the scale of q takes in log2 e, and its products with k would have more bits)
    how = dict(scale=1.0, cap=50.0, documents=docs)
    q, g, k, v = _normal(6, *shapes)
    q, k, g = q * np.float32(0.1), k * np.float32(0.1), g * np.float32(1e-3)
    q[..., 3] = np.where(np.arange(lq) % 3, 0, one)
    k[:, :, :, 3] = np.where(np.arange(130) % 5, 0, big)
    _near(_all(q, k, v, g, **how), nn_oracle.attention(q, k, v, dout=g, **how), names)
    q, g, k, v = _normal(7, *shapes)
    q, k, g = q * np.float32(0.1), k * np.float32(0.1), g * np.float32(1e-3)
    k[..., 3] = np.where(np.arange(130) % 3, 0, one)
    q[:, :, :, 3] = np.where(np.arange(lq) % 4, 0, big)
    _near(_all(q, k, v, g, **how)[:3], nn_oracle.attention(q, k, v, dout=g, **how), names[:3])
    q, g, k, v = _normal(8, *shapes)
    v[:, :, 77, 5], g[..., 5] = -big, 0
    _near(_all(q, k, v, g, documents=docs), nn_oracle.attention(q, k, v, dout=g, documents=docs), names)
    q, g, k, v = _normal(9, *shapes)
    g[:, 0, 2, 5], v[..., 5] = big, np.float32(2.0 ** -100)
    _near(_all(q, k, v, g, documents=docs), nn_oracle.attention(q, k, v, dout=g, documents=docs), names)


@pytest.mark.parametrize("lq", [5, 90])
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_rows_that_are_not_finite(lq, what):
    """A pair that counts gives NaN if its q or k is not finite, whatever sign their product has; rows beside it keep their values."""
    q, g, k, v = _normal(10, (2, 2, lq, 64), (2, 2, lq, 64), (2, 1, 130, 64), (2, 1, 130, 64))
    k = np.abs(k)
    docs = np.zeros((2, 130), np.int32)
    clean = nn_oracle.attention(q, k, v, documents=docs)
    q[0, 1, 3, 7] = what
    q[1, 0, 2] = what
    o, lse, dq, dk, dv = _all(q, k, v, g, documents=docs)
    bad = np.zeros((2, 2, lq), bool)
    bad[0, 1, 3] = bad[1, 0, 2] = True
    assert np.isnan(o[bad]).all() and np.isnan(lse[bad]).all() and np.isnan(dq[bad]).all()
    assert np.all(np.abs(o - clean["o"])[~bad] <= 2 * clean["o_off"][~bad]) and np.isfinite(lse[~bad]).all() and np.isfinite(dq[~bad]).all()
    # a row without keys does not look at what it holds
    o, lse, dq, dk, dv = _all(q, k, v, g, documents=docs, lengths=0)
    assert not (o.any() or dq.any() or dk.any() or dv.any()) and np.all(lse == -INF)


def test_rows_outside_the_sequence_belong_to_no_document():
    """Not to document 0 either: a key of document 0 that no row sees may hold anything, and its gradient is zero."""
    q, g, k, v = _normal(11, (1, 2, 60, 64), (1, 2, 60, 64), (1, 1, 100, 64), (1, 1, 100, 64))
    docs = np.ones((1, 100), np.int32)
    docs[0, 10:14], docs[0, 98:] = 0, 2
    how = dict(documents=docs, start=70)                  # rows at 70 to 129: 100 and 101 are outside, in a tile with documents 1 and 2
    want = nn_oracle.attention(q, k, v, dout=g, **how)
    k[0, 0, 10:14], v[0, 0, 12] = [[NAN], [INF], [-INF], [1.0]], NAN
    got = _all(q, k, v, g, **how)
    _near(got, want, ("o", "lse", "dq", "dk", "dv"))
    assert not got[3][0, 0, 10:14].any() and not got[4][0, 0, 10:14].any()


@pytest.mark.parametrize("lq", [1, 10, 33, 64, 200])
def test_keys_that_no_row_sees_have_no_gradient(lq):
    """Behind the last row, in front of the first one's document, behind the length: they may hold anything."""
    q, g, k, v = _normal(12, (2, 4, lq, 64), (2, 4, lq, 64), (2, 2, 300, 64), (2, 2, 300, 64))
    for how in (dict(causal=True, start=0), dict(causal=True, start=np.array([3, 50], np.int32)), dict(causal=True, start=2, cap=5.0, slopes=np.ones(4, np.float32))):
        want = nn_oracle.attention(q, k, v, dout=g, **how)
        hidden = k.copy(), v.copy()
        for b in range(2):
            last = lq + (how["start"] if np.ndim(how["start"]) == 0 else how["start"][b])
            hidden[0][b, :, last::2], hidden[0][b, :, last + 1::4], hidden[1][b, :, last:, 3] = NAN, INF, -INF
        got = _all(q, *hidden, g, **how)
        _near(got, want, ("o", "lse", "dq", "dk", "dv"))


def test_parameters_of_sampling_that_are_not_numbers():
    """NaN in an array of parameters, or as a uniform number, counts as 0."""
    rs = np.random.RandomState(12)
    logits = (rs.standard_normal((3, 700)) * 2).astype(np.float32)
    logits[:, ::2] = -INF
    nan, zero = dr.array(np.full(3, NAN)), dr.array(np.zeros(3, np.float32))
    dev, u = dr.array(logits), dr.array(np.array([0.1, 0.5, 0.99]))
    for name in ("temperature", "top_p", "min_p"):
        assert nn.sample(dev, u, **{name: nan}).get().tolist() == nn.sample(dev, u, **{name: zero}).get().tolist(), name
    assert nn.sample(dev, nan).get().tolist() == nn.sample(dev, zero).get().tolist()
    got = nn.sample(dev, u, temperature=dr.array(np.full(3, INF))).get()
    assert got.tolist() == [nn_oracle.sample(r, x, temperature=1e300) for r, x in zip(logits, (0.1, 0.5, 0.99))]


def test_sample_of_the_longest_rows():
    """2^25 tokens: each weight is a multiple of 2^-37 of the largest.  Equal ones share the range of the uniform
    numbers evenly; of two levels e^-3 apart the lower one's weight is off by less than 2^-33 of itself."""
    n = 1 << 25
    logits = np.zeros((1, n), np.float32)
    dev = dr.array(logits)
    for u in (0.0, 0.3, 0.75, 1 - 2.0 ** -26):
        assert nn.sample(dev, dr.array(np.array([u]))).get()[0] == int(u * n), u
    logits[0, :n // 2] = -3.0
    low = np.exp(-3.0)
    dev = dr.array(logits)
    for u in (0.02, 0.04, 0.3, 0.9):
        at = u * (n // 2) * (1 + low)
        want = at / low if at < n // 2 * low else n // 2 + at - n // 2 * low
        for got in (nn.sample(dev, dr.array(np.array([u]))).get()[0], nn.sample(dev, dr.array(np.array([u])), min_p=0.01).get()[0]):
            assert abs(got - want) <= 1 + n * 2.0 ** -32, (u, got, want)


def _in_a_program_with_torch(script):
    """A child process that imports torch first, as programs that use both do."""
    r = subprocess.run([sys.executable, "-u", "-c", textwrap.dedent(script)], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout[-1500:] + r.stderr[-3000:]


def test_writes_over_views_of_one_memory_taken_over_apart():
    """They read everything before they write, as those of one view do."""
    _in_a_program_with_torch("""
        import torch
        import numpy as np
        torch.zeros(1, device="cuda")
        import delayrepay_amd as dr
        n = 3000000
        for step in (1, 7, 100003):
            for up in (True, False):
                x = torch.arange(n, device="cuda", dtype=torch.float64)
                head, tail = dr.from_dlpack(x[:n - step]), dr.from_dlpack(x[step:])
                to, of = (tail, head) if up else (head, tail)
                want = np.arange(n, dtype=np.float64)
                for turn in range(3):
                    to[...] = of * 0.5 + 1.0
                    want[step if up else 0:n if up else n - step] = want[0 if up else step:n - step if up else n] * 0.5 + 1.0
                dr.synchronize()
                assert np.array_equal(x.cpu().numpy(), want), (step, up)
        x = torch.arange(40.0, device="cuda").view(4, 10)
        a, b = dr.from_dlpack(x[:, ::2]), dr.from_dlpack(x[:, 1::2])
        a[:, 1:] = a[:, :-1] + 100.0            # (its memory has elements of b in between)
        b[1:] = b[:-1] * -1.0
        c = dr.from_dlpack(x.t())
        c[...] = dr.from_dlpack(x).reshape((10, 4)) * 1.0
        want = np.arange(40.0, dtype=np.float32).reshape(4, 10)
        want[:, 2::2] = want[:, 0:-2:2] + 100
        want[1:, 1::2] = -want[:-1, 1::2]
        want.T[...] = want.reshape(10, 4).copy()
        dr.synchronize()
        assert np.array_equal(x.cpu().numpy(), want)
        print("done")
    """)


def test_what_is_computed_of_another_librarys_array_follows_its_writes():
    """An expression that is built again after the other library wrote is computed again."""
    _in_a_program_with_torch("""
        import torch
        import numpy as np
        torch.zeros(1, device="cuda")
        import delayrepay_amd as dr
        from delayrepay_amd import nn
        t = torch.arange(6.0, device="cuda").view(2, 3)
        a = dr.from_dlpack(t)
        held = a + 1.0
        first = held.get()
        kept = dr.array(np.ones((2, 3), np.float32))
        for turn in range(1, 4):
            before = [(a + 1.0).get(), (a * 2.0 + 3.0).sum(axis=1).get(), dr.sum(a).get(), (kept * a).get()]
            t += 10.0
            torch.cuda.synchronize()
            x = np.arange(6.0, dtype=np.float32).reshape(2, 3) + 10 * turn
            got = [(a + 1.0).get(), (a * 2.0 + 3.0).sum(axis=1).get(), dr.sum(a).get(), (kept * a).get(), ((a + 1.0) * 2.0).get()]
            for y, want in zip(got, (x + 1, (x * 2 + 3).sum(1), x.sum(), x, (x + 1) * 2)):
                assert np.allclose(y, want), (turn, y, want)
        x = torch.randn(1, 2, 40, 32, device="cuda")
        q = dr.from_dlpack(x)
        for _ in range(3):
            x.normal_()
            torch.cuda.synchronize()
            o = nn.attention(q * 2.0, q, q).get()
            s = torch.softmax(2 * x @ x.transpose(2, 3) / 32 ** 0.5, -1) @ x
            assert np.abs(o - s.cpu().numpy()).max() < 1e-5
        # this library's own writes are followed by what is held, as ever
        a[...] = 0.0
        assert np.array_equal(held.get(), np.ones((2, 3)))
        print("done")
    """)


def test_recorded_writes_over_views_of_one_memory():
    """Views taken over apart, disjoint columns among them: a replay does what the writes did."""
    _in_a_program_with_torch("""
        import torch
        import numpy as np
        torch.zeros(1, device="cuda")
        import delayrepay_amd as dr
        from delayrepay_amd import hip
        x = torch.arange(4000.0, device="cuda").view(40, 100)
        even, odd = dr.from_dlpack(x[:, ::2]), dr.from_dlpack(x[:, 1::2])
        with hip.record() as plan:
            even[...] = odd * 0.5
            odd[1:] = odd[:-1] + even[1:]
        dr.synchronize()
        want = np.arange(4000.0, dtype=np.float32).reshape(40, 100)

        def step():
            want[:, ::2] = want[:, 1::2] * np.float32(0.5)
            want[1:, 1::2] = want[:-1, 1::2] + want[1:, ::2]
        step()
        assert np.array_equal(x.cpu().numpy(), want)
        plan.as_graph()
        for turn in range(3):
            x += 1.0
            want += 1.0
            torch.cuda.synchronize()
            plan()
            dr.synchronize()
            step()
            assert np.array_equal(x.cpu().numpy(), want), turn
        print("done")
    """)
