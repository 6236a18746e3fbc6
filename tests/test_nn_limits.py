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
