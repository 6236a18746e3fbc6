"""`delayrepay.nn`: operators of language models that one fused expression cannot hold.

Softmax, norms and gated units are written as expressions and fuse (`e = exp(a - a.max(axis=-1,
keepdims=True)); e / e.sum(axis=-1, keepdims=True)`).  Not so attention, whose scores would go
through memory between its two products, rotary positions, which pair elements of a row, and
the drawing of a token, which selects by rank and by mass.  They are eager calls on arrays, as
`dot` is: lazy operands are evaluated first, the result is an array.

All sizes are read from the arrays: q (batch, heads, rows, size), k and v (batch, key heads, key
rows, size) with heads a multiple of key heads.  Any view will do (heads may lie behind rows in
memory); a view whose last axis is not dense is copied.  `out=` names arrays to write into,
in place of new ones.  Per-sequence arguments (`lengths`, `start` ...) are a number or an integer
array; what an array on the device holds cannot be checked and is clamped to the sizes.
"""
import math
import numbers

import numpy

from . import backend as be
from .delayarray import DelayArray, NPArray

_backend = be.backend
_ops = getattr(_backend, "operators", None)
_F32 = numpy.dtype(numpy.float32)
_F64 = numpy.dtype(numpy.float64)
_INTS = (numpy.dtype(numpy.int32), numpy.dtype(numpy.int64))

MAX_HEAD = 128           # elements of an attention head
MAX_ROTARY_HEAD = 512
_FAR = 1 << 30            # positions of rows are nearer to 0
_COUNTS = (-1, (1 << 31) - 1)
_LARGE = 2.0 ** 100       # scales and caps are smaller, and caps larger than its inverse: their products fit float32


# ---- arguments -------------------------------------------------------------------------------

def _array(x, name):
    if type(x) is NPArray:          # (the common kinds first, here and below: a short call is bound by its checks)
        return x.array
    if isinstance(x, DelayArray):
        return x._force()
    if _backend.is_ndarray(x):
        return x
    if isinstance(x, (numpy.ndarray, list, tuple)):
        return _backend.fallback.asarray(numpy.asarray(x))
    raise TypeError(f"{name} is an array, not a {type(x).__name__}")


def _floats(x, name, ndim, kinds=(_F32,)):
    x = _array(x, name)
    if x.dtype not in kinds:
        raise TypeError(f"{name} is {' or '.join(k.name for k in kinds)}, not {x.dtype} (convert it with astype)")
    if len(x.shape) != ndim:
        raise ValueError(f"{name} has {ndim} dimensions, not {len(x.shape)}")
    return x


def _shaped(x, name, shape):
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} has the shape {tuple(shape)}, not {tuple(x.shape)}")
    return x


def _integers(x, name, shape, number=True, within=_COUNTS):
    """None, a whole number, or an int32 array of `shape`: numbers of int64 arrays outside `within` are clamped to it,
    or without it all become others that are equal where they are."""
    if x is None:
        return None
    if type(x) is NPArray and x.dtype == _INTS[0] and x.shape == shape:
        return x.array
    if isinstance(x, (numbers.Integral, numpy.integer)) and not isinstance(x, (bool, numpy.bool_)):
        if not number:
            raise TypeError(f"{name} is an integer array")
        return int(x)
    x = _array(x, name)
    if x.dtype not in _INTS:
        raise TypeError(f"{name} holds int32 or int64, not {x.dtype}")
    _shaped(x, name, shape)
    return x if x.dtype == _INTS[0] else _ops.renumbered(x) if within is None else _ops.narrowed(x, *within)


def _number(x, name, low=-math.inf, above=False):
    if type(x) is float and low < x < math.inf:
        return x
    if isinstance(x, (bool, numpy.bool_)) or not isinstance(x, (numbers.Real, numpy.floating, numpy.integer)):
        raise TypeError(f"{name} is a number, not a {type(x).__name__}")
    x = float(x)
    if not math.isfinite(x) or x < low or (above and x == low):
        raise ValueError(f"{name} is a finite number {'above' if above else 'of at least'} {low:g}, not {x:g}"
                         if low > -math.inf else f"{name} is a finite number, not {x:g}")
    return x


def _targets(out, shapes, dtypes):
    """The arrays that `out` names, ready to be written to; Nones without it."""
    if out is None:
        return [None] * len(shapes)
    if type(out) is NPArray and len(shapes) == 1:
        arr = out.array
        if arr.shape == shapes[0] and arr.dtype is dtypes[0] and 0 not in getattr(arr, "_strides", (0,)):
            out._written()
            return [arr]
    outs = [out] if not isinstance(out, (tuple, list)) else list(out)
    if len(outs) != len(shapes):
        raise ValueError(f"out names {len(shapes)} array{'s' if len(shapes) > 1 else ''}, not {len(outs)}")
    arrays = []
    for i, (x, shape, dtype) in enumerate(zip(outs, shapes, dtypes)):
        name = "out" if len(outs) == 1 else "out[%d]" % i
        if type(x) is NPArray:
            arr = x.array
        elif isinstance(x, DelayArray):
            arr = x._force()
        elif _backend.is_ndarray(x):
            arr = x
        else:
            raise TypeError(f"{name} is an array, not a {type(x).__name__}")
        if arr.shape != shape:
            _shaped(arr, name, shape)
        if arr.dtype != dtype:
            raise TypeError(f"{name} is {dtype}, not {arr.dtype}")
        check = getattr(arr, "check_writable", None)
        if check is not None and arr.size:      # (an empty array has pitches of 0 by itself)
            check()
        arrays.append(arr)
    for x in outs:                    # (only once all of them are known to be right)
        if isinstance(x, DelayArray):
            x._written()
    return arrays


def _results(out, arrays):
    if out is not None:
        return out
    arrays = tuple(NPArray(a) for a in arrays)
    return arrays[0] if len(arrays) == 1 else arrays


# ---- attention -------------------------------------------------------------------------------

class _Mask:
    """Checked arguments that say which pairs count and how their scores are made."""

    __slots__ = ("scale", "causal", "start", "lengths", "prefix", "documents", "slopes", "cap", "plain")

    def __init__(self, q, k, scale, causal, start, lengths, prefix, documents, slopes, cap):
        batch, lk = k.shape[0], k.shape[2]
        # the common calls: no arguments but these, of them only `lengths` an array
        self.plain = prefix is None and documents is None and slopes is None and (start is None or type(start) is int) and type(lengths) is not int
        self.scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else _number(scale, "scale")
        if abs(self.scale) > _LARGE:
            raise ValueError(f"scale lies within 2**100 of 0, not at {self.scale:g}")
        if not isinstance(causal, (bool, numpy.bool_)):
            raise TypeError("causal is True or False")
        self.causal = bool(causal)
        self.cap = None if cap is None else _number(cap, "cap", 0.0, above=True)
        if cap is not None and not 1 / _LARGE <= self.cap <= _LARGE:
            raise ValueError(f"cap lies between 2**-100 and 2**100, not at {self.cap:g}")
        self.start = _integers(start, "start", (batch,), within=(-_FAR, _FAR))
        if isinstance(self.start, int) and abs(self.start) > _FAR:
            raise ValueError(f"start lies within 2**30 of 0, not at {self.start}")
        self.lengths = _integers(lengths, "lengths", (batch,))
        if self.plain:
            self.plain = not isinstance(self.lengths, int)
        if self.plain:
            self.prefix = self.documents = self.slopes = None
            return
        if isinstance(self.lengths, int) and not 0 <= self.lengths <= lk:
            raise ValueError(f"lengths lies in [0, {lk}], the rows of k, not {self.lengths}")
        self.prefix = _integers(prefix, "prefix", (batch,))
        if prefix is not None and not self.causal:
            raise ValueError("prefix belongs to causal attention: without causal=True every row sees every key")
        if isinstance(self.prefix, int) and self.prefix < 0:
            raise ValueError(f"prefix is at least 0, not {self.prefix}")
        self.slopes = None if slopes is None else _shaped(_floats(slopes, "slopes", 1), "slopes", (q.shape[1],))
        self.documents = _integers(documents, "documents", (batch, lk), number=False, within=None)


def _heads(q, k, v):
    q, k, v = _floats(q, "q", 4), _floats(k, "k", 4), _floats(v, "v", 4)
    (batch, hq, _, size), (kbatch, hkv, _, ksize) = q.shape, k.shape
    if tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"v has the shape of k, {tuple(k.shape)}, not {tuple(v.shape)}")
    if batch != kbatch or size != ksize:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or head size")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"the {hq} heads of q are not a multiple of the {hkv} of k")
    if not 1 <= size <= MAX_HEAD:
        raise ValueError(f"head sizes from 1 to {MAX_HEAD} are supported, not {size}")
    return q, k, v


def attention(q, k, v, *, scale=None, causal=False, start=None, lengths=None, prefix=None,
              documents=None, slopes=None, cap=None, with_lse=False, out=None):
    """softmax(scores) @ v for every head, in float32; the scores never go to memory.

    Scores are `scale * q @ k.T` (scale 1/sqrt(size)); with `cap`, cap * tanh(scores / cap); with
    `slopes` (heads,), less slopes[head] * |position of the row - position of the key|.

    Key j stands at position j and row i at `start` + i; the rows are the last ones of their
    sequence if `start` is not given.  A key counts for a row if j < `lengths` (all key rows
    without it), with `causal` if also j <= position of the row or j < `prefix`, and with
    `documents` (batch, key rows) if its document is the one at the row's position (rows outside the
    sequence have none).  A row without keys gives zeros.  Keys that do not count may hold anything, also
    what is not finite; a pair that counts gives NaN if its q or k is not finite.  `start` lies within 2**30
    of 0, `scale` within 2**100 of 0 and `cap` between 2**-100 and 2**100.  Sums are float32 and divided last: scores,
    and values times the number of keys, lie below 2**127; past that results are infinite or NaN.

    `with_lse` returns (output, lse): lse (batch, heads, rows), the logarithm of the sum of the
    exponentials of the scores (-inf for a row without keys), which `attention_grad` needs.

    One row and many, long caches and short: where the rows are few, blocks take ranges of the keys.
    batch * heads * (rows + 32) is below 2**28, and for more than 64 rows of a key head batch * key heads *
    (key rows + 32) as well (in the gradient both below 2**27).
    """
    q, k, v = _heads(q, k, v)
    how = _Mask(q, k, scale, causal, start, lengths, prefix, documents, slopes, cap)
    shapes = [q.shape] + ([q.shape[:3]] if with_lse else [])
    outs = _targets(out, shapes, [_F32] * len(shapes))
    return _results(out, _ops.attention(q, k, v, how, outs))


def attention_grad(dout, q, k, v, o, lse, *, scale=None, causal=False, start=None, lengths=None,
                   prefix=None, documents=None, slopes=None, cap=None, out=None):
    """(dq, dk, dv) of `attention` from the gradient of its output, its operands, output and lse.

    A key head's gradients are summed over the heads of q that share it.  The sums do not depend on
    timing: equal calls give equal bits.  `slopes` are constants.  What of the operands is not finite, or
    passes float32 in a sum, makes the gradients that it enters infinite or NaN.
    """
    q, k, v = _heads(q, k, v)
    dout = _shaped(_floats(dout, "dout", 4), "dout", q.shape)
    o = _shaped(_floats(o, "o", 4), "o", q.shape)
    lse = _shaped(_floats(lse, "lse", 3), "lse", q.shape[:3])
    how = _Mask(q, k, scale, causal, start, lengths, prefix, documents, slopes, cap)
    outs = _targets(out, [q.shape, k.shape, v.shape], [_F32] * 3)
    return _results(out, _ops.attention_grad(dout, q, k, v, o, lse, how, outs))


# ---- rotary positions ------------------------------------------------------------------------

class _Turn:
    """Checked arguments that say how pairs turn."""

    __slots__ = ("positions", "first", "frequencies", "base", "dims", "interleaved", "stretch", "magnitude", "weight", "eps")

    def __init__(self, x, positions, base, frequencies, dims, interleaved, stretch, magnitude, weight, eps):
        batch, heads, rows, size = x.shape
        if not 1 <= size <= MAX_ROTARY_HEAD:
            raise ValueError(f"head sizes from 1 to {MAX_ROTARY_HEAD} are supported, not {size}")
        if dims is None:
            dims = size - size % 2
        elif not isinstance(dims, (int, numpy.integer)) or isinstance(dims, bool) or dims % 2 or not 0 <= dims <= size:
            raise ValueError(f"dims is an even number of a head's {size} elements, not {dims!r}")
        self.dims = int(dims)
        self.positions, self.first = None, 0
        if type(positions) is int and -(1 << 52) < positions < 1 << 52:
            self.first = positions
        elif type(positions) is not NPArray and isinstance(positions, (numbers.Integral, numpy.integer)) and not isinstance(positions, (bool, numpy.bool_)):
            self.first = int(positions)
            if abs(self.first) >= 1 << 52:
                raise ValueError("positions lie below 2**52")
        else:
            p = _array(positions, "positions")
            if p.dtype not in _INTS:
                raise TypeError(f"positions holds int32 or int64, not {p.dtype}")
            if tuple(p.shape) not in ((rows,), (batch, rows)):
                raise ValueError(f"positions has the shape {(rows,)} or {(batch, rows)}, not {tuple(p.shape)}")
            self.positions = p
        self.base = base if type(base) is float and 0.0 < base < math.inf else _number(base, "base", 0.0, above=True)
        self.frequencies = None
        if frequencies is not None:
            f = _array(frequencies, "frequencies")
            if f.dtype != _F64:
                raise TypeError(f"frequencies is float64, not {f.dtype}")
            self.frequencies = _shaped(f, "frequencies", (self.dims // 2,))
        if not isinstance(interleaved, (bool, numpy.bool_)):
            raise TypeError("interleaved is True or False")
        self.interleaved = bool(interleaved)
        self.stretch = stretch if type(stretch) is float and 0.0 < stretch < math.inf else _number(stretch, "stretch", 0.0, above=True)
        self.magnitude = magnitude if type(magnitude) is float and abs(magnitude) < math.inf else _number(magnitude, "magnitude")
        self.eps = eps if type(eps) is float and 0.0 <= eps < math.inf else _number(eps, "eps", 0.0)
        self.weight = None
        if weight is not None:
            w = _array(weight, "weight")
            if w.dtype != x.dtype:
                raise TypeError(f"weight has the type of the rows, {x.dtype}, not {w.dtype}")
            if tuple(w.shape) not in ((size,), (heads, size)):
                raise ValueError(f"weight has the shape {(size,)} or {(heads, size)}, not {tuple(w.shape)}")
            self.weight = w


def rotary(x, positions, *, base=10000.0, frequencies=None, dims=None, interleaved=False,
           stretch=1.0, magnitude=1.0, weight=None, eps=1e-6, out=None):
    """Rows of x (batch, heads, rows, size) turned by their positions, float32 or float64.

    Pair number i of the first `dims` elements (all of them if not given) turns by the angle
    position * frequency_i / stretch: elements (i, i + dims/2), or neighbours (2i, 2i + 1) with
    `interleaved`.  Frequencies are base ** (-2 i / dims), or a float64 array (dims/2,); `stretch`
    scales positions for contexts longer than those trained on, `magnitude` multiplies the turned
    elements.  `positions` is an integer array (rows,) or (batch, rows), or the first row's position.
    Angles are computed in 64 bits (positions of an int64 array beyond 2**53 are rounded).

    With `weight`, (size,) or (heads, size), each row is first divided by the root of (the mean of its
    squares + eps) and multiplied by the weight: the norm of queries and keys in the same pass.  Squares, eps and
    magnitude are numbers of the rows' type: elements of float32 rows lie below 2**59, of float64 ones below 2**507.
    """
    x = _floats(x, "x", 4, (_F32, _F64))
    how = _Turn(x, positions, base, frequencies, dims, interleaved, stretch, magnitude, weight, eps)
    outs = _targets(out, [x.shape], [x.dtype])
    return _results(out, _ops.rotary(x, how, outs))


def rotary_grad(dy, x, positions, *, base=10000.0, frequencies=None, dims=None, interleaved=False,
                stretch=1.0, magnitude=1.0, weight=None, eps=1e-6, out=None):
    """Gradient of `rotary` from that of its result: dx without a weight (x is not used and may be
    None), (dx, dweight) with one.  Equal calls give equal bits."""
    dy = _floats(dy, "dy", 4, (_F32, _F64))
    how = _Turn(dy, positions, base, frequencies, dims, interleaved, stretch, magnitude, weight, eps)
    if weight is None:
        outs = _targets(out, [dy.shape], [dy.dtype])
        return _results(out, _ops.rotary_grad(dy, None, how, outs))
    x = _shaped(_floats(x, "x", 4, (dy.dtype,)), "x", dy.shape)
    outs = _targets(out, [dy.shape, how.weight.shape], [dy.dtype] * 2)
    return _results(out, _ops.rotary_grad(dy, x, how, outs))


# ---- tokens ----------------------------------------------------------------------------------

def sample(logits, uniforms, *, temperature=1.0, top_k=None, top_p=None, min_p=None, out=None):
    """One token for each row of logits (batch, vocabulary), int64, drawn with given numbers.

    Weights are exp(logit / temperature).  `top_k` keeps the k largest (of equal ones the lower
    numbers), `top_p` of these the first whose weights reach that part of their sum, `min_p` of these the
    ones of at least that part of the largest.  The token is the first one, by number, at which the
    kept weights summed up exceed uniforms[row] (in [0, 1): `random.device().random(batch)`) of their sum.
    A temperature of 0 takes the largest; they go up to float32's largest.  Each of the four is a number or an array (batch,), float32 or
    (top_k) integers, in which a top_k below 1 stands for all, numbers out of range for the nearest in it and NaN for 0.
    A logit that is NaN or -inf is never drawn; a row without another gives -1.

    Sums are whole numbers of 62 bits: the token depends on no order of summation.  A weight is a multiple of 2**-s of
    the largest, s = 62 - (bits of the vocabulary) but at most 52 (45 for 128000 tokens); what is smaller than
    half of that is none, vocabulary * 2**-(s + 1) of the largest at most in all (2**-29, and 2**-7 for 2**28 tokens).
    """
    logits = _floats(logits, "logits", 2)
    batch, vocabulary = logits.shape
    if not 1 <= vocabulary < 1 << 28:
        raise ValueError(f"vocabularies of 1 to 2**28 tokens are supported, not {vocabulary}")
    uniforms = _shaped(_floats(uniforms, "uniforms", 1, (_F32, _F64)), "uniforms", (batch,))

    def part(x, name, none, low, high, above):
        if x is None:
            return none
        if type(x) is float and low < x <= high:
            return x
        if isinstance(x, (numbers.Real, numpy.floating, numpy.integer)) and not isinstance(x, bool):
            x = float(x)
            if not low <= x <= high or (above and x == low):
                raise ValueError(f"{name} lies in {'(' if above else '['}{low:g}, {high:g}], not at {x:g}")
            return x
        return _shaped(_floats(x, name, 1), name, (batch,))
    temperature = part(temperature, "temperature", 1.0, 0.0, 3.4028234663852886e38, False)
    top_p = part(top_p, "top_p", 1.0, 0.0, 1.0, True)
    min_p = part(min_p, "min_p", 0.0, 0.0, 1.0, False)
    top_k = _integers(top_k, "top_k", (batch,))
    if isinstance(top_k, int) and top_k < 1:
        raise ValueError(f"top_k is at least 1, not {top_k}")
    outs = _targets(out, [(batch,)], [numpy.dtype(numpy.int64)])
    return _results(out, _ops.sample(logits, uniforms, temperature, 0 if top_k is None else top_k, top_p, min_p, outs))
