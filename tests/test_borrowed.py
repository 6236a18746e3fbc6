"""Memory of another library: what a fused write does with it, on arrays whose addresses are made up (nothing is launched)."""
import numpy as np
import pytest

from delayrepay_amd import hip
from delayrepay_amd.devarray import Borrowed, ndarray


def _taken(at, n, dtype=np.float32, strides=(1,)):
    """A 1-d array over made-up memory at the address `at`."""
    return ndarray((n,), dtype, Borrowed(((n - 1) * strides[0] + 1) * np.dtype(dtype).itemsize, at, None), 0, strides)


def _plan(dst, *leaves):
    tracer = hip.Tracer()
    refs = [tracer.leaf(a) for a in leaves]
    root = refs[0] if len(refs) == 1 else tracer.op("add", refs[0][1], refs[0][1], [r[0] for r in refs])
    return hip._plan_write(tracer, root, dst)


@pytest.mark.parametrize("ahead,hazard", [(4, True), (-4, True), (0, True), (396, True), (400, False), (-400, False), (1 << 20, False)])
def test_views_of_one_memory_taken_over_apart(ahead, hazard):
    """A kernel that writes one and reads the other goes through another allocation where their bytes overlap."""
    base = 1 << 33
    dst = _taken(base, 100)
    assert _plan(dst, _taken(base + ahead, 100)).hazard == hazard
    assert _plan(dst, _taken(base + (1 << 30), 100), _taken(base + ahead, 100)).hazard == hazard
    assert not _plan(dst, dst).hazard                     # (the very same view is read where it is written)


def test_types_and_pitches_of_overlapping_views():
    base = 1 << 33
    assert _plan(_taken(base, 10, np.float64), _taken(base + 76, 10)).hazard
    assert not _plan(_taken(base, 10, np.float64), _taken(base + 80, 10)).hazard
    assert _plan(_taken(base, 10, strides=(3,)), _taken(base + 108, 10)).hazard
    assert not _plan(_taken(base, 10, strides=(3,)), _taken(base + 112, 10)).hazard
    assert not _plan(hip.placeholder((100,), np.float32), _taken(base, 100)).hazard


def test_only_the_view_is_copied_back(monkeypatch):
    """What stands between the elements of a view belongs to the other library: no copy passes over it."""
    fired, base, shadow = [], 1 << 33, 1 << 34
    monkeypatch.setattr(hip, "_fire", lambda plan, outs: fired.append((plan, outs)))
    monkeypatch.setattr(hip.hiprt, "malloc", lambda nbytes: shadow)
    monkeypatch.setattr(hip.hiprt, "memcpy_d2d", lambda *args: pytest.fail("a copy of the whole span"))
    whole = _taken(base, 10, strides=(3,))
    dst, src = whole[1:], whole[:-1]
    hip._write(_plan(dst, src), dst)
    whole.buf.shadow = None
    (first, to_shadow), (second, to_memory) = fired
    assert first.hazard and to_shadow == [shadow + 12] and [a.ptr for a in first.leaves] == [base]
    assert not second.hazard and to_memory == [base + 12]
    assert [(a.ptr, a.shape, a._strides) for a in second.leaves] == [(shadow + 12, (9,), (3,))]
    assert whole.buf.ptr == base and whole.buf.version > 0
