"""The operators of `nn` on the device: packs their argument structs (include/drhip.h), holds
workspaces from the pool, and gives results their place."""
import math

import numpy

from . import hip, hiprt
from .devarray import Buffer, ndarray

_F32 = numpy.dtype(numpy.float32)


def _dense(x):
    """The array, copied if its last axis is not dense (or an index array not dense at all)."""
    return x.copy() if x.shape[-1] > 1 and x._strides[-1] != 1 else x


def _strides(x):
    return x._strides[:3]


def _ptr(x):
    return 0 if x is None else x.ptr


def _reach(x):
    """First and last byte that the array can touch, as addresses."""
    lo, hi = hip._extent(x)
    at, item = x.buf.ptr, x.dtype.itemsize
    return at + lo * item, at + hi * item


def _apart(x, others):
    """Whether `x` shares no memory with the others."""
    a, n = x.buf.ptr, x.buf.nbytes
    for y in others:
        if y is None or not y.size or not x.size:
            continue
        if a < y.buf.ptr + y.buf.nbytes and y.buf.ptr < a + n:
            lo, hi = _reach(x)
            ylo, yhi = _reach(y)
            if lo < yhi and ylo < hi:
                return False
    return True


def _places(outs, shapes, dtype, used, same=None):
    """Arrays to compute into: the ones asked for, or new ones where those are not dense
    in their last axis or share memory with an operand (`same`: one that may be exactly the output)."""
    places = []
    for i, (out, shape) in enumerate(zip(outs, shapes)):
        direct = out is not None and not (out.shape and out.shape[-1] > 1 and out._strides[-1] != 1)
        if direct:
            others = used + [o for n, o in enumerate(outs) if n != i]
            if same is not None and out._strides == same._strides and out.ptr == same.ptr:
                others = [u for u in others if u is not same]
            direct = _apart(out, others)
        places.append(out if direct else ndarray(shape, dtype))
    return places


def _give(outs, places):
    for out, place in zip(outs, places):
        if out is not None and out is not place:
            hip.assign(out, place)
    return [place if out is None else out for out, place in zip(outs, places)]


def _contiguous(x):
    return x if x is None or x.is_contiguous else x.copy()


def _run(func, packer, fields, ints, work, used, written):
    """Call one operator with `work` bytes of workspace between its two runs of fields."""
    buf = None
    if work:
        buf = Buffer(work)
    args = packer.pack(*fields, buf.ptr if buf else 0, work, *ints)
    hip.issue_operator(func, args, used + written + ([buf] if buf else []), written)


def _attention_args(q, k, v, o, lse, dout, grads, how):
    def index(x):
        return _contiguous(x) if isinstance(x, ndarray) else None
    lengths, start, prefix = how.lengths, how.start, how.prefix
    if isinstance(lengths, int):       # a number: the rows behind it do not exist
        k, v = k[:, :, :lengths], v[:, :, :lengths]
    arrays = [index(lengths), index(start), index(prefix),
              None if how.documents is None else _dense(how.documents),
              None if how.slopes is None else _contiguous(how.slopes)]
    if isinstance(lengths, int) and arrays[3] is not None:
        arrays[3] = arrays[3][:, :lengths]
    none = (0, 0, 0)
    fields = (q.ptr, k.ptr, v.ptr, o.ptr, _ptr(lse), _ptr(dout), *[_ptr(g) for g in grads], *[_ptr(x) for x in arrays])
    lk = k.shape[2]
    far = (1 << 31) - 1
    ints = (*_strides(q), *_strides(k), *_strides(v), *_strides(o),
            *(none if dout is None else _strides(dout)), *[s for g in grads for s in (none if g is None else _strides(g))],
            0 if arrays[3] is None else arrays[3]._strides[0],
            q.shape[0], q.shape[1], k.shape[1], q.shape[2], lk, q.shape[3], int(how.causal),
            0 if start is None else 1, max(-far, min(far, start)) if isinstance(start, int) else 0,
            min(prefix, lk) if isinstance(prefix, int) else 0,
            how.scale, how.cap or 0.0)
    return fields, ints, [x for x in arrays if x is not None]


def attention(q, k, v, how, outs):
    q, k, v = _dense(q), _dense(k), _dense(v)
    masks = [how.documents, how.slopes] + [x for x in (how.lengths, how.start, how.prefix) if isinstance(x, ndarray)]
    shapes = [q.shape, q.shape[:3]][:len(outs)]
    places = _places(outs, shapes, _F32, [q, k, v] + masks)
    if len(places) > 1 and not places[1].is_contiguous:
        places[1] = ndarray(shapes[1], _F32)
    o, lse = places[0], places[1] if len(places) > 1 else None
    fields, ints, arrays = _attention_args(q, k, v, o, lse, None, (None, None, None), how)
    probe = hiprt.ATTENTION.pack(*fields, 0, 0, *ints)
    _run(hiprt.attention, hiprt.ATTENTION, fields, ints, hiprt.attention_work(probe, False), [q, k, v] + arrays, places)
    return _give(outs, places)


def attention_grad(dout, q, k, v, o, lse, how, outs):
    dout, q, k, v, o, lse = _dense(dout), _dense(q), _dense(k), _dense(v), _dense(o), _contiguous(lse)
    used = [dout, q, k, v, o, lse]
    masks = [how.documents, how.slopes] + [x for x in (how.lengths, how.start, how.prefix) if isinstance(x, ndarray)]
    places = _places(outs, [q.shape, k.shape, v.shape], _F32, used + masks)
    grads = list(places)
    if isinstance(how.lengths, int):       # the rows behind it have no gradient
        grads[1:] = [g[:, :, :how.lengths] for g in grads[1:]]
        for g in places[1:]:
            if how.lengths < k.shape[2]:
                hip.assign(g[:, :, how.lengths:], 0.0)
    fields, ints, arrays = _attention_args(q, k, v, o, lse, dout, grads, how)
    probe = hiprt.ATTENTION.pack(*fields, 0, 0, *ints)
    _run(hiprt.attention_grad, hiprt.ATTENTION, fields, ints, hiprt.attention_work(probe, True), used + arrays, places)
    return _give(outs, places)


def _rotary(x, how, outs, sign, dy=None):
    rows = dy if x is None else x
    batch, heads, count, size = rows.shape
    weight = None if how.weight is None else _dense(how.weight)
    per_head = weight is not None and len(weight.shape) == 2
    positions = None if how.positions is None else _dense(how.positions)
    frequencies = None if how.frequencies is None else _contiguous(how.frequencies)
    used = [a for a in (x, dy, weight, positions, frequencies) if a is not None]
    grad = dy is not None and x is not None
    shapes = [rows.shape] + ([weight.shape] if grad else [])
    # a row is read whole before it is written: the result may take an operand's place
    places = _places(outs, shapes, rows.dtype, used, same=dy if grad else rows)
    if grad and not places[1].is_contiguous:
        places[1] = ndarray(shapes[1], rows.dtype)
    none = (0, 0, 0)
    fields = (rows.ptr, places[0].ptr, _ptr(weight), dy.ptr if grad else 0, places[1].ptr if grad else 0, _ptr(positions), _ptr(frequencies))
    ints = (*_strides(rows), *_strides(places[0]), *(_strides(dy) if grad else none),
            weight._strides[0] if per_head else 0,
            positions._strides[0] if positions is not None and len(positions.shape) == 2 else 0, how.first,
            -2.0 * math.log2(how.base) / max(how.dims, 1), 1.0 / how.stretch, how.magnitude, sign, how.eps,
            batch, heads, count, size, how.dims, (size + 3) // 4 * 4,
            int(how.interleaved), int(rows.dtype.itemsize == 8),
            int(positions is not None and positions.dtype.itemsize == 8))
    work = hiprt.rotary_work(hiprt.ROTARY.pack(*fields, 0, 0, *ints)) if grad else 0
    _run(hiprt.rotary, hiprt.ROTARY, fields, ints, work, used, places)
    return _give(outs, places)


def rotary(x, how, outs):
    return _rotary(_dense(x), how, outs, 1.0)


def rotary_grad(dy, x, how, outs):
    return _rotary(None if x is None else _dense(x), how, outs, -1.0, _dense(dy))


def sample(logits, uniforms, temperature, top_k, top_p, min_p, outs):
    logits, uniforms = _dense(logits), _contiguous(uniforms)
    batch, vocabulary = logits.shape

    def either(x):
        return (_contiguous(x), 0) if isinstance(x, ndarray) else (None, x)
    (t, t_all), (k, k_all), (p, p_all), (m, m_all) = (either(x) for x in (temperature, top_k, top_p, min_p))
    used = [x for x in (logits, uniforms, t, k, p, m) if x is not None]
    places = _places(outs, [(batch,)], numpy.dtype(numpy.int64), used)
    one = 2.0 ** min(52, 62 - max(1, (vocabulary - 1).bit_length()))      # (float64 holds it)
    args = hiprt.SAMPLE.pack(logits.ptr, uniforms.ptr, places[0].ptr, _ptr(t), _ptr(p), _ptr(m), _ptr(k), logits._strides[0],
                             t_all, p_all, m_all, one, min(k_all, vocabulary), batch, vocabulary, int(uniforms.dtype.itemsize == 8))
    hip.issue_operator(hiprt.sample, args, used + places, places)
    return _give(outs, places)
