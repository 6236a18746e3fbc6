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
