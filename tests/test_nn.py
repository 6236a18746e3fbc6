"""`nn` without a GPU: its formulas under `DELAY_CPU` against the oracle (in a child process, the backend
being chosen at import), the oracle's gradients against differences, and refusals on either backend."""
import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest

from oracle import nn_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _child(script, **env):
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(script)], cwd=ROOT, capture_output=True, text=True,
                       env={**os.environ, **env}, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    return r.stdout


def test_formulas_on_the_numpy_backend():
    _child("""
        import numpy as np
        import delayrepay as dnp
        from oracle import nn_oracle
        assert dnp.backend.__name__.endswith(".cpu")
        rs = np.random.RandomState(1)
        f = lambda *s: rs.standard_normal(s).astype(np.float32)
        docs = np.array([[1, 1, 2, 2, 2, 3, 3, 3, 3], [5, 5, 5, 5, 4, 4, 9, 9, 1]], np.int32)
        cases = [dict(), dict(causal=True), dict(causal=True, lengths=np.array([4, 0], np.int32)), dict(causal=True, prefix=3, cap=2.0),
                 dict(causal=True, start=np.array([-2, 3], np.int64), slopes=f(4) ** 2), dict(causal=True, documents=docs),
                 dict(lengths=5, scale=0.3, documents=docs)]
        for how in cases:
            q, k, v, g = f(2, 4, 6, 8), f(2, 2, 9, 8), f(2, 2, 9, 8), f(2, 4, 6, 8)
            if how.get("lengths") is not None:       # rows behind a sequence may hold anything
                n = np.broadcast_to(how["lengths"], (2,))
                for b in range(2):
                    k[b, :, n[b]:], v[b, :, n[b]:] = np.nan, np.inf
            want = nn_oracle.attention(q, k, v, dout=g, **how)
            dev = [dnp.array(x) for x in (q, k, v, g)]
            o, lse = dnp.nn.attention(*dev[:3], with_lse=True, **how)
            grads = dnp.nn.attention_grad(dev[3], *dev[:3], o, lse, **how)
            for name, got in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *grads)):
                got = got.get()
                assert got.dtype == np.float32
                with np.errstate(invalid="ignore"):
                    assert np.all((got == want[name]) | (np.abs(got - want[name]) <= want[name + "_off"])), (how, name)
        for how in (dict(), dict(interleaved=True, dims=6, stretch=4.0), dict(weight=f(3, 10)), dict(weight=f(10), dims=4, magnitude=1.3, base=500.0),
                    dict(frequencies=np.array([1.0, 0.1]), dims=4)):
            x, g = f(2, 3, 5, 10), f(2, 3, 5, 10)
            at = rs.randint(0, 100000, (2, 5))
            dx = {k: dnp.array(v) if isinstance(v, np.ndarray) else v for k, v in how.items()}
            assert np.allclose(dnp.nn.rotary(dnp.array(x), at, **dx).get(), nn_oracle.rotary(x, at, **how), rtol=1e-6, atol=1e-6)
            got = dnp.nn.rotary_grad(dnp.array(g), dnp.array(x), at, **dx)
            want = nn_oracle.rotary(x, at, dy=g, **how)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert np.allclose(a.get(), b, rtol=1e-5, atol=1e-5)
        logits = np.round(f(50, 40) * 3) / 2          # (many ties)
        logits[3], logits[4, 7], logits[5, 2] = -np.inf, np.nan, np.inf
        u = rs.rand(50)
        for how in (dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.7), dict(min_p=0.2, temperature=1.4), dict(top_k=9, top_p=0.8, min_p=0.05)):
            got = dnp.nn.sample(dnp.array(logits), dnp.array(u), **how).get()
            want = [nn_oracle.sample(r, x, **how) for r, x in zip(logits, u)]
            assert got.dtype == np.int64 and got.tolist() == want, how
        # results in the arrays asked for, and what was computed from these before is computed again
        out = dnp.array(np.zeros((2, 4, 6, 8), np.float32))
        twice = out * 2
        assert not twice.get().any()
        assert dnp.nn.attention(*dev[:3], out=out, causal=True) is out and out.get().any()
        assert np.array_equal(twice.get(), out.get() * 2, equal_nan=True)
        assert np.array_equal(dnp.from_dlpack(np.arange(4.0)).get(), np.arange(4.0))
    """, DELAY_CPU="1")


@pytest.mark.parametrize("how", [dict(), dict(causal=True, cap=1.5), dict(causal=True, prefix=2, slopes=np.array([0.3, 0.1])),
                                 dict(causal=True, lengths=np.array([5, 3]), documents=np.array([[1, 1, 2, 2, 2, 2], [1, 1, 1, 2, 2, 2]]))])
def test_the_oracle_gradients_agree_with_differences(how):
    rs = np.random.RandomState(2)
    q, k, v, g = (rs.standard_normal(s) for s in ((2, 2, 4, 3), (2, 1, 6, 3), (2, 1, 6, 3), (2, 2, 4, 3)))
    want = nn_oracle.attention(q, k, v, dout=g, **how)
    step = 1e-6          # central differences: off by about step^2 and 1e-16 / step
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        for _ in range(12):
            at = tuple(rs.randint(0, n) for n in x.shape)
            keep = x[at]
            x[at] = keep + step
            up = (nn_oracle.attention(q, k, v, **how)["o"] * g).sum()
            x[at] = keep - step
            down = (nn_oracle.attention(q, k, v, **how)["o"] * g).sum()
            x[at] = keep
            assert abs((up - down) / (2 * step) - want[name][at]) < 1e-7


def test_the_oracle_rotary_gradients_agree_with_differences():
    rs = np.random.RandomState(3)
    x, g, w = rs.standard_normal((1, 2, 3, 6)), rs.standard_normal((1, 2, 3, 6)), rs.standard_normal((2, 6))
    how = dict(dims=4, interleaved=True, magnitude=1.2)
    dx, dw = nn_oracle.rotary(x, 7, weight=w, dy=g, **how)
    step = 1e-6
    for name, y, want in (("x", x, dx), ("w", w, dw)):
        for at in np.ndindex(y.shape):
            keep = y[at]
            y[at] = keep + step
            up = (nn_oracle.rotary(x, 7, weight=w, **how) * g).sum()
            y[at] = keep - step
            down = (nn_oracle.rotary(x, 7, weight=w, **how) * g).sum()
            y[at] = keep
            assert abs((up - down) / (2 * step) - want[at]) < 1e-7, name


REFUSALS = """
    import numpy as np
    import delayrepay as dnp
    from delayrepay_amd import nn

    if dnp.backend.__name__.endswith(".cpu"):
        make = dnp.array
    else:              # arrays without device memory: every refusal comes before the device is asked
        from delayrepay_amd.devarray import placeholder
        make = lambda x: dnp.NPArray(placeholder(x.shape, x.dtype))
    f = lambda *s, t=np.float32: make(np.zeros(s, t))
    i = lambda *s, t=np.int32: make(np.zeros(s, t))
    q, k = f(2, 4, 3, 8), f(2, 2, 5, 8)
    lse = f(2, 4, 3)

    def refused(kind, word, call, *args, **kwargs):
        try:
            call(*args, **kwargs)
        except kind as e:
            assert word in str(e), (word, str(e))
        else:
            raise AssertionError(("not refused", word))

    A, G = nn.attention, nn.attention_grad
    refused(TypeError, "float32", A, f(2, 4, 3, 8, t=np.float64), k, k)
    refused(TypeError, "float32", A, i(2, 4, 3, 8), k, k)
    refused(TypeError, "array", A, 3.0, k, k)
    refused(ValueError, "dimensions", A, f(4, 3, 8), k, k)
    refused(ValueError, "shape of k", A, q, k, f(2, 2, 6, 8))
    refused(ValueError, "differ", A, q, f(1, 2, 5, 8), f(1, 2, 5, 8))
    refused(ValueError, "differ", A, q, f(2, 2, 5, 9), f(2, 2, 5, 9))
    refused(ValueError, "multiple", A, q, f(2, 3, 5, 8), f(2, 3, 5, 8))
    refused(ValueError, "multiple", A, q, f(2, 0, 5, 8), f(2, 0, 5, 8))
    refused(ValueError, "head sizes", A, f(1, 1, 3, 129), f(1, 1, 3, 129), f(1, 1, 3, 129))
    refused(ValueError, "head sizes", A, f(1, 1, 3, 0), f(1, 1, 3, 0), f(1, 1, 3, 0))
    refused(ValueError, "prefix belongs", A, q, k, k, prefix=2)
    refused(ValueError, "prefix", A, q, k, k, prefix=-1, causal=True)
    refused(ValueError, "lengths", A, q, k, k, lengths=6)
    refused(ValueError, "lengths", A, q, k, k, lengths=i(3))
    refused(TypeError, "lengths", A, q, k, k, lengths=f(2))
    refused(TypeError, "lengths", A, q, k, k, lengths=True)
    refused(TypeError, "start", A, q, k, k, start=1.5)
    refused(ValueError, "documents", A, q, k, k, documents=i(2, 4))
    refused(TypeError, "documents", A, q, k, k, documents=1)
    refused(ValueError, "slopes", A, q, k, k, slopes=f(2))
    refused(ValueError, "cap", A, q, k, k, cap=0.0)
    refused(ValueError, "cap", A, q, k, k, cap=float("inf"))
    refused(ValueError, "cap lies", A, q, k, k, cap=1e-50)
    refused(ValueError, "cap lies", A, q, k, k, cap=1e35)
    refused(ValueError, "scale lies", A, q, k, k, scale=-1e39)
    refused(ValueError, "start lies", A, q, k, k, start=1 << 31)
    refused(ValueError, "scale", A, q, k, k, scale=float("nan"))
    refused(TypeError, "causal", A, q, k, k, causal=1)
    refused(ValueError, "out", A, q, k, k, out=f(2, 4, 3, 9))
    refused(TypeError, "out", A, q, k, k, out=f(2, 4, 3, 8, t=np.float64))
    refused(TypeError, "out", A, q, k, k, out=[3])
    refused(ValueError, "out names 2", A, q, k, k, out=q, with_lse=True)
    refused(ValueError, "lse", G, q, q, k, k, q, f(2, 4, 4))
    refused(ValueError, "dout", G, f(2, 4, 2, 8), q, k, k, q, lse)
    refused(ValueError, "out names 3", G, q, q, k, k, q, lse, out=q)
    R = nn.rotary
    refused(ValueError, "head sizes", R, f(1, 1, 2, 513), 0)
    refused(ValueError, "dims", R, q, 0, dims=3)
    refused(ValueError, "dims", R, q, 0, dims=10)
    refused(TypeError, "positions", R, q, f(3))
    refused(TypeError, "positions", R, q, 1.0)
    refused(ValueError, "positions", R, q, i(4))
    refused(ValueError, "positions", R, q, 1 << 60)
    refused(ValueError, "stretch", R, q, 0, stretch=0.0)
    refused(TypeError, "weight", R, q, 0, weight=f(8, t=np.float64))
    refused(ValueError, "weight", R, q, 0, weight=f(3, 8))
    refused(TypeError, "frequencies", R, q, 0, frequencies=f(4))
    refused(ValueError, "frequencies", R, q, 0, frequencies=f(3, t=np.float64))
    refused(TypeError, "interleaved", R, q, 0, interleaved=1)
    refused(ValueError, "eps", R, q, 0, eps=-1.0)
    refused(ValueError, "x has the shape", nn.rotary_grad, q, k, 0, weight=f(8))
    refused(TypeError, "x is an array", nn.rotary_grad, q, None, 0, weight=f(8))
    S = nn.sample
    logits, u = f(2, 9), f(2)
    refused(TypeError, "logits", S, f(2, 9, t=np.float64), u)
    refused(ValueError, "logits", S, f(9), u)
    refused(ValueError, "vocabularies", S, f(2, 0), u)
    refused(ValueError, "uniforms", S, logits, f(3))
    refused(ValueError, "temperature", S, logits, u, temperature=-1.0)
    refused(ValueError, "temperature", S, logits, u, temperature=float("nan"))
    refused(ValueError, "top_k", S, logits, u, top_k=0)
    refused(TypeError, "top_k", S, logits, u, top_k=2.0)
    refused(ValueError, "top_p", S, logits, u, top_p=0.0)
    refused(ValueError, "top_p", S, logits, u, top_p=1.1)
    refused(ValueError, "min_p", S, logits, u, min_p=-0.1)
    refused(ValueError, "min_p", S, logits, u, min_p=f(3))
    refused(TypeError, "out", S, logits, u, out=f(2))
    print("all refused")
"""


@pytest.mark.parametrize("cpu", [False, True])
def test_refusals(cpu):
    env = {"DELAY_CPU": "1"} if cpu else {}
    assert "all refused" in _child(REFUSALS, **env)


def test_the_library_refuses_what_its_launches_cannot_hold():
    """The C entry points check sizes by themselves (before a device is asked for, where one is not needed)."""
    import ctypes
    from delayrepay_amd import hiprt

    def attention(batch=1, hq=2, hkv=1, lq=3, lk=3, d=8, prefix=0, scale=1.0, cap=0.0, grad=1):
        args = hiprt.ATTENTION.pack(*[0] * 15, 0, *[0] * 25, batch, hq, hkv, lq, lk, d, 0, 0, 0, prefix, scale, cap)
        n = ctypes.c_uint64()
        return hiprt.lib().drhip_attention_work(args, grad, ctypes.byref(n))

    def rotary(batch=1, heads=2, rows=3, d=8, dims=8, pad=8):
        args = hiprt.ROTARY.pack(*[0] * 8, 0, *[0] * 12, 0.0, 1.0, 1.0, 1.0, 0.0, batch, heads, rows, d, dims, pad, 0, 0, 0)
        n = ctypes.c_uint64()
        return hiprt.lib().drhip_rotary_work(args, ctypes.byref(n))
    assert attention() == 0 and rotary() == 0
    for bad in (dict(hq=3, hkv=2), dict(d=129), dict(d=0), dict(lq=-1), dict(lk=1 << 28), dict(batch=1 << 23), dict(batch=1 << 20, lq=1 << 20), dict(prefix=-1), dict(batch=1 << 21),
                dict(scale=1e38), dict(scale=float("nan")), dict(cap=1e-38), dict(cap=float("inf"))):
        assert attention(**bad) == 20002, bad
    assert attention(batch=1 << 21, grad=0) == 0          # (fewer matrices to pack)
    for bad in (dict(d=513, pad=516), dict(dims=7), dict(dims=10), dict(pad=6), dict(rows=-1), dict(batch=1 << 20, rows=1 << 20)):
        assert rotary(**bad) == 20002, bad


def test_argument_structs_have_the_size_of_the_header(tmp_path):
    """The packed bytes are read as C structs: none shorter than its struct, fillings at the end included."""
    from delayrepay_amd import hiprt
    source, program = tmp_path / "sizes.c", tmp_path / "sizes"
    source.write_text('#include <stdio.h>\n#include "drhip.h"\nint main(void) { printf("%zu %zu %zu", sizeof(drhip_attention_t), sizeof(drhip_rotary_t), sizeof(drhip_sample_t)); return 0; }\n')
    subprocess.run(["cc", "-I", os.path.join(ROOT, "include"), "-o", str(program), str(source)], check=True)
    sizes = [int(x) for x in subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [a.size + b.size for a, b in ((hiprt.ATTENTION_HEAD, hiprt.ATTENTION_TAIL), (hiprt.ROTARY_HEAD, hiprt.ROTARY_TAIL), (hiprt.SAMPLE_HEAD, hiprt.SAMPLE_TAIL))]
    assert sizes[:2] == [hiprt.ATTENTION.size, hiprt.ROTARY.size]
