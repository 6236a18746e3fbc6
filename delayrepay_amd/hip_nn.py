"""The operators of `nn` on the device: packs their argument structs (include/drhip.h), holds
workspaces from the pool, and gives results their place."""
import math

import numpy

from . import hip, hiprt
from .devarray import Buffer, ndarray

_F32, _I64 = numpy.dtype(numpy.float32), numpy.dtype(numpy.int64)


def narrowed(x, low, high):
    """The int64 array (one dimension) in int32, with its numbers clamped to [low, high]."""
    out = ndarray(x.shape, numpy.int32)
    if x.size:
        hip.issue_operator(hiprt.clamp, hiprt.CLAMP.pack(x.ptr, out.ptr, x._strides[0], x.size, low, high), [x, out], [out])
    return out


def _dense(x):
    """The array, copied if its last axis is not dense."""
    return x if x._strides[-1] == 1 or x.shape[-1] <= 1 else x.copy()


def renumbered(x):
    """An int32 array of numbers that are equal within a row where those of the int64 array are."""
    x = _dense(x)
    batch, n = x.shape
    out = ndarray(x.shape, numpy.int32)
    if x.size:
        slots = 1 << (2 * n - 1).bit_length()
        table = Buffer(batch * slots * 4)
        hip.issue_operator(hiprt.renumber, hiprt.RENUMBER.pack(x.ptr, out.ptr, table.ptr, x._strides[0], batch, n, slots), [x, out, table], [out])
    return out


def _strides(x):
    return x._strides[:3]


def _steps(x):
    return None if x is None else x._strides


def _ptr(x):
    return 0 if x is None else x.buf.ptr + x.offset * x.dtype.itemsize


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
    if len(outs) == 1 and outs[0] is not None and outs[0]._strides[-1] == 1:       # (the common call first)
        a, n = outs[0].buf.ptr, outs[0].buf.nbytes
        for y in used:
            if y is not None and a < y.buf.ptr + y.buf.nbytes and y.buf.ptr < a + n:
                break
        else:
            return [outs[0]]
    places = []
    for i, (out, shape) in enumerate(zip(outs, shapes)):
        if out is None:
            places.append(ndarray(shape, dtype))
            continue
        direct = not (out.shape[-1] > 1 and out._strides[-1] != 1)
        if direct:
            others = used if len(outs) == 1 else used + [o for n, o in enumerate(outs) if n != i]
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


# What depends on geometry and options alone -> (its part of the argument struct, workspace bytes).  Addresses are
# not part of it, and no workspace is kept.
_PLANS = {}
_PLANS_MAX = 1024


def _remember(key, plan):
    if len(_PLANS) >= _PLANS_MAX:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


def _plan(key, head, tail, fields, make, work_of):
    """The remembered plan, or a new one: `make()` gives the tail's fields, work_of(args) the workspace."""
    plan = _PLANS.get(key)
    if plan is None:
        packed = tail.pack(*make())
        plan = _remember(key, (packed, work_of(head.pack(*fields, 0, 0) + packed)))
    return plan


def _run(func, head, fields, plan, used, written):
    """Call one operator, with a workspace from the pool where it needs one."""
    tail, work = plan
    if work:
        buf = Buffer(work)
        hip.issue_operator(func, head.pack(*fields, buf.ptr, work) + tail, used + written + [buf], written)
    else:
        hip.issue_operator(func, head.pack(*fields, 0, 0) + tail, used + written, written)


_NONE = (0, 0, 0)


def _attention(func, grad, q, k, v, o, lse, dout, grads, how, used, written):
    def index(x):
        return _contiguous(x) if isinstance(x, ndarray) else None
    lengths, start, prefix = how.lengths, how.start, how.prefix
    if how.plain and not grad:         # (the same with less to do: a short call is bound by this)
        if lengths is not None:
            lengths = _contiguous(lengths)
            used = used + [lengths]
        fields = (q.ptr, k.ptr, v.ptr, o.ptr, 0 if lse is None else lse.ptr, 0, 0, 0, 0, 0 if lengths is None else lengths.ptr, 0, 0, 0, 0)
        plain = (q.shape, q._strides, k.shape, k._strides, v._strides, o._strides, how.causal, "last" if start is None else start, how.scale, how.cap)
        plan = _PLANS.get(plain)
        if plan is not None:
            return _run(func, hiprt.ATTENTION_HEAD, fields, plan, used, written)
    if isinstance(lengths, int):       # a number: the rows behind it do not exist
        k, v = k[:, :, :lengths], v[:, :, :lengths]
    documents = None if how.documents is None else _dense(how.documents)
    if isinstance(lengths, int) and documents is not None:
        documents = documents[:, :lengths]
    arrays = [index(lengths), index(start), index(prefix), documents, None if how.slopes is None else _contiguous(how.slopes)]
    fields = (q.ptr, k.ptr, v.ptr, o.ptr, _ptr(lse), _ptr(dout), *[_ptr(g) for g in grads], *[_ptr(x) for x in arrays])
    key = (func, q.shape, q._strides, k.shape, k._strides, v._strides, o._strides, _steps(dout),
           *[_steps(g) for g in grads], _steps(documents), how.causal,
           start if isinstance(start, int) else "last" if start is None else "array", prefix if isinstance(prefix, int) else None, how.scale, how.cap)

    def make():
        lk = k.shape[2]
        return (*_strides(q), *_strides(k), *_strides(v), *_strides(o),
                *(_NONE if dout is None else _strides(dout)), *[s for g in grads for s in (_NONE if g is None else _strides(g))],
                0 if documents is None else documents._strides[0],
                q.shape[0], q.shape[1], k.shape[1], q.shape[2], lk, q.shape[3], int(how.causal),
                0 if start is None else 1, start if isinstance(start, int) else 0,
                min(prefix, lk) if isinstance(prefix, int) else 0,
                how.scale, how.cap or 0.0)
    plan = _plan(key, hiprt.ATTENTION_HEAD, hiprt.ATTENTION_TAIL, fields, make, lambda args: hiprt.attention_work(args, grad))
    if how.plain and not grad:
        _remember(plain, plan)
    _run(func, hiprt.ATTENTION_HEAD, fields, plan, used + [x for x in arrays if x is not None], written)


def attention(q, k, v, how, outs):
    q, k, v = _dense(q), _dense(k), _dense(v)
    operands = [q, k, v]
    if how.plain:
        operands.append(how.lengths)
    else:
        operands += [how.documents, how.slopes] + [x for x in (how.lengths, how.start, how.prefix) if isinstance(x, ndarray)]
    shapes = [q.shape, q.shape[:3]][:len(outs)]
    places = _places(outs, shapes, _F32, operands)
    if len(places) > 1 and not places[1].is_contiguous:
        places[1] = ndarray(shapes[1], _F32)
    _attention(hiprt.attention, False, q, k, v, places[0], places[1] if len(places) > 1 else None, None, (None, None, None), how, [q, k, v], places)
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
    _attention(hiprt.attention_grad, True, q, k, v, o, lse, dout, grads, how, used, places)
    return _give(outs, places)


def _rotary(x, how, outs, sign, dy=None):
    rows = dy if x is None else x
    batch, heads, count, size = rows.shape
    weight = None if how.weight is None else _dense(how.weight)
    per_head = weight is not None and len(weight.shape) == 2
    if per_head and heads != 1 and weight._strides[0] == 0:       # (a pitch of 0 is the sign of one weight for all)
        weight = weight.copy()
    positions = None if how.positions is None else _dense(how.positions)
    frequencies = None if how.frequencies is None else _contiguous(how.frequencies)
    used = [a for a in (x, dy, weight, positions, frequencies) if a is not None]
    grad = dy is not None and x is not None
    shapes = [rows.shape, weight.shape] if grad else [rows.shape]
    # a row is read whole before it is written: the result may take an operand's place
    places = _places(outs, shapes, rows.dtype, used, same=dy if grad else rows)
    if grad and not places[1].is_contiguous:
        places[1] = ndarray(shapes[1], rows.dtype)
    fields = (rows.ptr, places[0].ptr, 0 if weight is None else weight.ptr, dy.ptr if grad else 0, places[1].ptr if grad else 0,
              0 if positions is None else positions.ptr, 0 if frequencies is None else frequencies.ptr)
    key = (grad, sign, rows.shape, rows._strides, places[0]._strides, dy._strides if grad else None, rows.dtype.itemsize, per_head and weight._strides,
           None if positions is None else (positions.shape, positions._strides, positions.dtype.itemsize),
           how.first, how.base, how.dims, how.stretch, how.magnitude, how.eps, how.interleaved)

    def make():
        return (*_strides(rows), *_strides(places[0]), *(_strides(dy) if grad else _NONE),
                weight._strides[0] if per_head else 0,
                positions._strides[0] if positions is not None and len(positions.shape) == 2 else 0, how.first,
                -2.0 * math.log2(how.base) / max(how.dims, 1), 1.0 / how.stretch, how.magnitude, sign, how.eps,
                batch, heads, count, size, how.dims, (size + 3) // 4 * 4,
                int(how.interleaved), int(rows.dtype.itemsize == 8),
                int(positions is not None and positions.dtype.itemsize == 8))
    plan = _plan(key, hiprt.ROTARY_HEAD, hiprt.ROTARY_TAIL, fields, make, hiprt.rotary_work)
    _run(hiprt.rotary, hiprt.ROTARY_HEAD, fields, plan, used, places)
    return _give(outs, places)


def rotary(x, how, outs):
    return _rotary(_dense(x), how, outs, 1.0)


def rotary_grad(dy, x, how, outs):
    return _rotary(None if x is None else _dense(x), how, outs, -1.0, _dense(dy))


def sample(logits, uniforms, temperature, top_k, top_p, min_p, outs):
    logits, uniforms = _dense(logits), _contiguous(uniforms)
    batch, vocabulary = logits.shape
    used, places_of = [logits, uniforms], [0, 0, 0, 0]
    numbers = (temperature, top_p, min_p, top_k)
    if ndarray in (type(temperature), type(top_p), type(min_p), type(top_k)):
        arrays = [_contiguous(x) if isinstance(x, ndarray) else None for x in numbers]
        numbers = tuple(0 if isinstance(x, ndarray) else x for x in numbers)
        places_of = [_ptr(x) for x in arrays]
        used += [x for x in arrays if x is not None]
    places = _places(outs, [(batch,)], _I64, used)
    key = (logits._strides[0], batch, vocabulary, uniforms.dtype.itemsize, numbers)
    tail = _PLANS.get(key)
    if tail is None:
        t, p, m, k = numbers
        one = 2.0 ** min(52, 62 - max(1, (vocabulary - 1).bit_length()))      # (float64 holds it)
        tail = hiprt.SAMPLE_TAIL.pack(logits._strides[0], t, p, m, one, min(k, vocabulary), batch, vocabulary, int(uniforms.dtype.itemsize == 8))
        _remember(key, tail)
    args = hiprt.SAMPLE_HEAD.pack(logits.ptr, uniforms.ptr, places[0].ptr, *places_of) + tail
    hip.issue_operator(hiprt.sample, args, used + places, places)
    return _give(outs, places)
