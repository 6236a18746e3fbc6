"""`nn` under `DELAY_CPU` at the ends of its arguments' ranges, and limits that the library checks by itself
(no GPU: the NumPy backend in a child process, the library's checks without a device)."""
import os
import subprocess
import sys
import textwrap

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _child(script, **env):
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(script)], cwd=ROOT, capture_output=True, text=True,
                       env={**os.environ, **env}, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    return r.stdout


def test_numbers_of_64_bits_are_clamped():
    """Numbers that int32 does not hold count as the nearest in range, not as their low 32 bits."""
    _child("""
        import numpy as np
        import delayrepay as dnp
        rs = np.random.RandomState(1)
        q, k, v = (dnp.array(rs.standard_normal(s).astype(np.float32)) for s in ((4, 2, 3, 8), (4, 2, 9, 8), (4, 2, 9, 8)))
        wide = np.array([2 ** 63 - 1, 2 ** 32 + 3, -2 ** 63, -2 ** 32 + 3])
        for how, same in ((dict(lengths=wide), [9, 9, 0, 0]), (dict(prefix=wide, causal=True), [9, 9, 0, 0]),
                          (dict(start=wide, causal=True), [2 ** 30, 2 ** 30, -2 ** 30, -2 ** 30])):
            name = next(iter(how))
            got = dnp.nn.attention(q, k, v, **how).get()
            want = dnp.nn.attention(q, k, v, **dict(how, **{name: np.array(same, np.int32)})).get()
            assert np.array_equal(got, want), name
        logits, u = dnp.array(rs.standard_normal((4, 50)).astype(np.float32)), dnp.array(rs.rand(4))
        assert dnp.nn.sample(logits, u, top_k=wide).get().tolist() == dnp.nn.sample(logits, u).get().tolist()
    """, DELAY_CPU="1")


def test_documents_of_64_bits():
    """Numbers that agree in their low 32 bits are different documents."""
    _child("""
        import numpy as np
        import delayrepay as dnp
        rs = np.random.RandomState(2)
        q, k, v = (dnp.array(rs.standard_normal(s).astype(np.float32)) for s in ((2, 2, 5, 8), (2, 2, 9, 8), (2, 2, 9, 8)))
        order = rs.randint(0, 3, (2, 9))
        ids = np.array([1, 1 + 2 ** 32, -2 ** 63 + 1])[order]
        got, want = (dnp.nn.attention(q, k, v, documents=x).get() for x in (ids, order.astype(np.int32)))
        assert np.array_equal(got, want)
    """, DELAY_CPU="1")


def test_the_library_checks_the_table_of_renumbered_documents():
    from delayrepay_amd import hiprt
    for batch, n, slots in ((-1, 3, 8), (1, -1, 8), (1, 3, 4), (1, 3, 7), (1, 0, 1), (1, 1 << 28, 1 << 29), (1 << 23, 3, 8), (1, 3, -8)):
        assert hiprt.lib().drhip_renumber(hiprt.RENUMBER.pack(16, 16, 16, n, batch, n, slots)) == 20002, (batch, n, slots)


def test_the_library_checks_what_it_clamps():
    from delayrepay_amd import hiprt
    for n, low, high in ((-1, 0, 1), (1 << 28, 0, 1), (3, 2, 1)):
        assert hiprt.lib().drhip_clamp(hiprt.CLAMP.pack(16, 16, 1, n, low, high)) == 20002, (n, low, high)


def test_argument_structs_have_the_size_of_the_header(tmp_path):
    from delayrepay_amd import hiprt
    source, program = tmp_path / "sizes.c", tmp_path / "sizes"
    source.write_text('#include <stdio.h>\n#include "drhip.h"\nint main(void) { printf("%zu %zu", sizeof(drhip_renumber_t), sizeof(drhip_clamp_t)); return 0; }\n')
    subprocess.run(["cc", "-I", os.path.join(ROOT, "include"), "-o", str(program), str(source)], check=True)
    sizes = subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in sizes] == [hiprt.RENUMBER.size, hiprt.CLAMP.size]


def test_caches_that_fit_the_device_are_not_refused():
    """Blocks are counted by key heads, and only where keys are packed."""
    import ctypes
    from delayrepay_amd import hiprt

    def work(batch, hq, hkv, lq, lk, d=128, grad=0):
        args = hiprt.ATTENTION.pack(*[0] * 15, 0, *[0] * 25, batch, hq, hkv, lq, lk, d, 1, 0, 0, 0, 1.0, 0.0)
        n = ctypes.c_uint64()
        return hiprt.lib().drhip_attention_work(args, grad, ctypes.byref(n)), n.value
    for batch, hq, hkv, lk in ((64, 64, 8, 65536), (64, 32, 8, 131072), (32, 64, 8, 131072), (256, 32, 8, 131072), (1 << 20, 2, 1, 3000), (1, 1, 1, (1 << 28) - 1)):
        rc, n = work(batch, hq, hkv, 1, lk)
        assert rc == 0 and n < 1 << 30, (batch, hq, hkv, lk)
    assert work(64, 64, 8, 128, 65536)[0] == 0 and work(16, 64, 8, 128, 65536, grad=1)[0] == 0        # (bounds by heads of q refused both)
    # what does not fit one launch still is
    for bad in (dict(batch=64, hq=64, hkv=64, lq=128, lk=65536), dict(batch=64, hq=64, hkv=32, lq=1, lk=65536, grad=1), dict(batch=1 << 13, hq=64, hkv=1, lq=512, lk=8)):
        assert work(**bad)[0] == 20002, bad


def test_rotary_counts_the_threads_of_its_launch():
    """2^32 threads and more are refused by the library itself, fewer are not."""
    import ctypes
    from delayrepay_amd import hiprt

    def work(batch, heads, rows, d):
        args = hiprt.ROTARY.pack(*[0] * 8, 0, *[0] * 12, 0.0, 1.0, 1.0, 1.0, 0.0, batch, heads, rows, d, d, d, 0, 0, 0)
        n = ctypes.c_uint64()
        return hiprt.lib().drhip_rotary_work(args, ctypes.byref(n))
    # heads of 264 take 64 lanes, for two heads where there are many: 2^27 of them are 2^32 threads
    assert work(1, 8, 1 << 24, 264) == 20002 and work(1, 8, (1 << 24) - 4, 264) == 0
    assert work(1, 1, 1 << 26, 264) == 20002 and work(1, 1, (1 << 26) - 4, 264) == 0
    assert work(4, 1, 1 << 26, 8) == 0 and work(1 << 20, 1 << 19, 1 << 20, 8) == 20002
    assert work(1 << 16, 1, 1 << 16, 8) == 20002


def test_pairs_that_are_not_finite():
    """A pair that counts gives NaN if its q or k is not finite, whatever sign their product has."""
    _child("""
        import numpy as np
        import delayrepay as dnp
        rs = np.random.RandomState(3)
        q, k, v, g = (rs.standard_normal(s).astype(np.float32) for s in ((1, 1, 4, 8), (1, 1, 6, 8), (1, 1, 6, 8), (1, 1, 4, 8)))
        k = np.abs(k)

        def run(q, k):
            dev = [dnp.array(x) for x in (q, k, v, g)]
            o, lse = dnp.nn.attention(*dev[:3], causal=True, start=0, with_lse=True)
            return [x.get()[0, 0] for x in (o, lse, *dnp.nn.attention_grad(dev[3], *dev[:3], o, lse, causal=True, start=0))]
        clean = run(q, k)
        for what in (np.inf, -np.inf, np.nan):
            bad = q.copy()
            bad[0, 0, 1, 3] = what
            o, lse, dq, dk, dv = run(bad, k)
            assert np.isnan(o[1]).all() and np.isnan(lse[1]) and np.isnan(dq[1]).all()
            for x, y in zip((o, lse, dq), clean):
                assert np.array_equal(np.delete(x, 1, 0), np.delete(y, 1, 0))
            assert np.isnan(dk[:2]).any()
            for x, y in zip((dk, dv), clean[3:]):          # (sums in 64 bits in another order, rounded to 32)
                assert np.allclose(x[2:], y[2:], rtol=2.0 ** -23, atol=1e-12)
            bad = k.copy()
            bad[0, 0, 2, 5] = what
            o, lse, dq, dk, dv = run(q, bad)
            assert np.isnan(o[2:]).all() and np.array_equal(o[:2], clean[0][:2]) and np.array_equal(dq[:2], clean[2][:2])
    """, DELAY_CPU="1")


def test_parameters_of_sampling_that_are_not_numbers():
    """NaN counts as 0, an infinite temperature as the largest: neither draws what has no weight."""
    _child("""
        import numpy as np
        import delayrepay as dnp
        from oracle import nn_oracle
        rs = np.random.RandomState(4)
        logits = (rs.standard_normal((3, 70)) * 2).astype(np.float32)
        logits[:, ::2], logits[1, 1] = -np.inf, np.nan
        f = lambda x: dnp.array(np.full(3, x, np.float32))
        u = dnp.array(np.array([0.1, 0.5, 0.99]))
        for name in ("temperature", "top_p", "min_p"):
            got, want = (dnp.nn.sample(dnp.array(logits), u, **{name: f(x)}).get().tolist() for x in (np.nan, 0.0))
            assert got == want, name
        assert dnp.nn.sample(dnp.array(logits), f(np.nan)).get().tolist() == dnp.nn.sample(dnp.array(logits), f(0.0)).get().tolist()
        got = dnp.nn.sample(dnp.array(logits), u, temperature=f(np.inf)).get()
        assert got.tolist() == [nn_oracle.sample(r, x, temperature=1e300) for r, x in zip(logits, (0.1, 0.5, 0.99))]
    """, DELAY_CPU="1")


def test_keys_that_do_not_count_take_no_memory():
    """What is not finite is added row by row: 1500 rows and keys of 64 would otherwise take 1.1 GB for each product."""
    _child("""
        import resource
        import numpy as np
        import delayrepay as dnp
        rs = np.random.RandomState(5)
        q, k, v, g = (rs.standard_normal((1, 1, 1500, 64)).astype(np.float32) for _ in range(4))
        args = dict(causal=True, start=-700)
        dev = [dnp.array(x) for x in (q, k, v, g)]
        dnp.nn.attention(*dev[:3], **args)
        before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
        clean = dnp.nn.attention(*dev[:3], with_lse=True, **args)
        clean = [*clean, *dnp.nn.attention_grad(dev[3], *dev[:3], *clean, **args)]
        k[:, :, 800:], v[:, :, 800:] = np.nan, np.inf
        dev = [dnp.array(x) for x in (q, k, v, g)]
        got = dnp.nn.attention(*dev[:3], with_lse=True, **args)
        got = [*got, *dnp.nn.attention_grad(dev[3], *dev[:3], *got, **args)]
        for x, y in zip(got, clean):
            assert np.allclose(x.get(), y.get(), rtol=2.0 ** -23, atol=1e-12)
        assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 500 << 10
        v[0, 0, 5, 3], v[0, 0, 6, 3], v[0, 0, 9, 4] = np.inf, -np.inf, np.nan
        o = dnp.nn.attention(*dev[:2], dnp.array(v), **args).get()[0, 0]
        assert np.isfinite(o[:705]).all() and np.all(o[705, 3] == np.inf) and np.isnan(o[706:, 3]).all() and np.isnan(o[709:, 4]).all()
        assert np.isfinite(o[:709, 4]).all() and np.isfinite(np.delete(o, [3, 4], 1)).all()
    """, DELAY_CPU="1")


def test_a_lost_part_of_the_products_would_be_noticed():
    """What the GPU test of attention's precision allows lies between products of three bfloat16 parts and those of two."""
    import numpy as np
    from tests import nn_precision as p
    for size in p.SIZES:
        x = p.inputs(*size)
        want = p.attention(*x, p.plain_product, np.float64)
        plain, three, two = ({n: p.error(y, want[n]) for n, y in p.attention(*x, product).items()}
                             for product in (p.plain_product, p.split_product(3), p.split_product(2)))
        for n in want:
            assert three[n] <= 1.5 * plain[n] and two[n] >= 3 * p.WORST * plain[n], (size, n, plain[n], three[n], two[n])
