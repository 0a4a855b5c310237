"""Operators over the rows of a matrix: layer normalisation, embedding lookup and distillation from a
teacher's top logits, each with its gradient.

They are what a language model runs around its matrix products, and extend the statistics and reductions
of this layer (mean/var: dpnp/tensor/_statistical_functions.py:38-270; logsumexp:
dpnp/tensor/_reduction.py:515-577), which compute the same values in many launches.  Conventions are the
reductions' own: arrays of one queue, results allocated on it in C order, ``out`` of exactly the result's
shape and type (computed in a temporary first where it partly overlaps an input).  Data is float16, float32
or float64; sums and statistics are float32, or float64 for float64 data, and every result is rounded once.

The kernels walk rows of unit stride whose starts lie at most two strides apart; an array of any other layout
is copied into such a one first.
"""

from __future__ import annotations

import numbers

import numpy as np

from .. import _lib
from ..memory import ExecutionPlacementError
from . import _tensor_impl as ti
from . import _tensor_rows_impl as tri
from ._copy_utils import _empty, astype
from ._elementwise_common import _common_queue
from ._manipulation_functions import normalize_axis_tuple, permute_dims, reshape
from ._usmarray import usm_ndarray

_HALF, _SINGLE, _DOUBLE = np.dtype("f2"), np.dtype("f4"), np.dtype("f8")
_ACCUMULATION = {_HALF: _SINGLE, _SINGLE: _SINGLE, _DOUBLE: _DOUBLE}
_INDEX = (np.dtype("i4"), np.dtype("i8"))


# ------------------------------------------------------------------------------------------- arguments
def _check_array(x, what):
    if not isinstance(x, usm_ndarray):
        raise TypeError(f"{what}: expected dpnp.tensor.usm_ndarray, got {type(x)}")
    return x


def _accumulation_type(x, what):
    try:
        return _ACCUMULATION[x._dtype]
    except KeyError:
        raise TypeError(f"{what}: float16, float32 or float64 is needed, got {x._dtype}") from None


def _execution_queue(*arrays):
    q = _common_queue([a._queue for a in arrays if a is not None])
    if q is None:
        raise ExecutionPlacementError("Execution placement can not be unambiguously inferred from input arguments.")
    return q


def _number(value, what):
    if isinstance(value, (bool, np.bool_)) or not isinstance(value, numbers.Real):
        raise TypeError(f"{what}: a real number is needed, got {type(value)}")
    return float(value)


def _walkable(shape, strides):
    """Whether the kernels can walk the rows: unit stride along the last axis and, with the leading axes
    merged where they follow one another, at most two strides between the starts."""
    if not shape:
        return False
    if shape[-1] > 1 and strides[-1] != 1:
        return False
    levels, stride = 0, 0
    for ext, st in zip(shape[:-1], strides[:-1]):
        if ext == 1:
            continue
        if levels and stride == st * ext:
            stride = st
            continue
        levels += 1
        stride = st
    return levels <= 2


def _dense(x, q):
    """`x` itself when it is C-contiguous, else a copy that is."""
    if x._flags & _lib.FLAG_C:
        return x
    res = _empty(x._shape, x._dtype, q)
    ti._copy_usm_ndarray_into_usm_ndarray(x, res, q)
    return res


def _rows(x, q):
    return x if (x._flags & _lib.FLAG_C) or _walkable(x._shape, x._strides) else _dense(x, q)


def _typed(x, dt, q):
    """`x` as a C-contiguous array of type `dt`."""
    return _dense(x if x._dtype == dt else astype(x, dt, order="C"), q)


class _Out:
    """Where one result goes.  ``target``: the caller's array, checked against the result's shape and type,
    or None; ``buf``: what the kernel writes -- the target itself where it can be written directly (C order,
    or rows that can be walked; no overlap with an input, other than being exactly one of `in_place`),
    otherwise a new array."""

    __slots__ = ("buf", "target", "direct")

    def __init__(self, target, shape, dtype, q, inputs, in_place=(), walkable=False, allocate=True):
        self.target = target
        self.direct = False
        if target is not None:
            if not target._flags & _lib.FLAG_W:
                raise ValueError("provided `out` array is read-only")
            if target._shape != shape:
                raise ValueError("The shape of input and output arrays are inconsistent. "
                                 f"Expected output shape is {shape}, got {target._shape}")
            if target._dtype != dtype:
                raise ValueError(f"Output array of type {dtype} is needed, got {target._dtype}")
            if _common_queue((q, target._queue)) is None:
                raise ExecutionPlacementError("Input and output allocation queues are not compatible")
            if any(ext > 1 and st == 0 for ext, st in zip(target._shape, target._strides)):
                raise ValueError("Memory addressed by the output array is not sufficiently ample.")
            self.direct = bool(target._flags & _lib.FLAG_C) or (walkable and _walkable(shape, target._strides))
            for x in inputs:
                if self.direct and x is not None and ti._array_overlap(x, target):
                    self.direct = any(x is y for y in in_place) and ti._same_logical_tensors(x, target)
        self.buf = target if self.direct else _empty(shape, dtype, q) if allocate else None

    def finish(self, q):
        """The caller's result, once the kernel has been queued."""
        if self.target is None:
            return self.buf
        if not self.direct:
            ti._copy_usm_ndarray_into_usm_ndarray(self.buf, self.target, q)
        return self.target


def _unpack_out(out, count, what):
    """`out` of an operator with several results: None, or a tuple with an array or None for each; the ranges of
    memory of the arrays must not overlap."""
    if out is None:
        return (None,) * count
    if not isinstance(out, (tuple, list)) or len(out) != count:
        raise TypeError(f"{what}: `out` must be a tuple of {count} arrays (or None)")
    for o in out:
        if o is not None and not isinstance(o, usm_ndarray):
            raise TypeError(f"output array must be of usm_ndarray type, got {type(o)}")
    for i, a in enumerate(out):
        for b in out[:i]:
            if a is not None and b is not None and ti._array_overlap(a, b):
                raise ValueError("Arrays index overlapping segments of memory")
    return tuple(out)


# ------------------------------------------------------------------------------------------- direct route
# A call whose arrays are C-contiguous and live on one queue object goes to the library as it is: the types and
# shapes that results are allocated from are compared here, everything else is checked by the library, and
# whatever it refuses takes the general route below, which copies what has to be copied and words the refusal.
# (As for the elementwise functions, the general route is the specification.)
_nat = tri._nat
_new = usm_ndarray._new_dense


def _plain(q, *arrays):
    """Whether all arrays (None: absent) are C-contiguous and on the queue `q`."""
    for a in arrays:
        if a is not None and (type(a) is not usm_ndarray or a._queue is not q or not a._flags & _lib.FLAG_C):
            return False
    return True


def _plain_rows(q, *arrays):
    """The same for arrays of rows, which may lie apart."""
    for a in arrays:
        if a is not None and (type(a) is not usm_ndarray or a._queue is not q
                              or not (a._flags & _lib.FLAG_C or _walkable(a._shape, a._strides))):
            return False
    return True


def _core(a):
    return None if a is None else a._core()


def _outs(out, count):
    """`out` of an operator with `count` results as that many entries; None when it is something else."""
    if out is None:
        return (None,) * count
    if count == 1:
        return (out,)
    return out if type(out) is tuple and len(out) == count else None


def _weights_fit(x, *weights):
    """Weights of the last axis, all of one type that goes with x."""
    dt = None
    for w in weights:
        if w is None:
            continue
        if w._shape != x._shape[-1:] or (dt is not None and w._dtype != dt):
            return False
        dt = w._dtype
    return dt is None or dt == x._dtype or (dt == _SINGLE and x._dtype == _HALF)


def _direct_layer_norm(x, weight, bias, eps, return_stats, out):
    outs = _outs(out, 3 if return_stats else 1)
    if outs is None or type(x) is not usm_ndarray or type(eps) is not float or not 0 <= eps < float("inf") or not x._shape:
        return None
    q, acc = x._queue, _ACCUMULATION.get(x._dtype)
    if acc is None or x._shape[-1] == 0 or not _plain_rows(q, x, outs[0]) or not _plain(q, weight, bias, *outs[1:]) \
            or not _weights_fit(x, weight, bias):
        return None
    y = _new(x._shape, x._dtype, q) if outs[0] is None else outs[0]
    mean = rstd = None
    if return_stats:
        lead = x._shape[:-1]
        mean = _new(lead, acc, q) if outs[1] is None else outs[1]
        rstd = _new(lead, acc, q) if outs[2] is None else outs[2]
    try:
        _nat.layer_norm(x._core(), _core(weight), _core(bias), eps, y._core(), _core(mean), _core(rstd), q._stream)
    except (TypeError, ValueError):
        return None
    return (y, mean, rstd) if return_stats else y


def _direct_layer_norm_backward(dy, x, mean, rstd, weight, weight_grads, out):
    outs = _outs(out, 3)
    if outs is None or type(x) is not usm_ndarray or not x._shape or not weight_grads:
        return None
    if dy is None or mean is None or rstd is None:
        return None
    q = x._queue
    if not _plain_rows(q, x, dy, outs[0]) or not _plain(q, mean, rstd, weight, *outs[1:]) or x._dtype not in _ACCUMULATION or x._shape[-1] == 0:
        return None
    if dy._shape != x._shape or dy._dtype != x._dtype or mean._shape != x._shape[:-1] or not _weights_fit(x, weight):
        return None
    dx, dw, db = outs
    if weight is None and (dw is not None or db is not None):
        return None
    wt = x._dtype if weight is None else weight._dtype
    dx = _new(x._shape, x._dtype, q) if dx is None else dx
    dw = _new(x._shape[-1:], wt, q) if dw is None else dw
    db = _new(x._shape[-1:], wt, q) if db is None else db
    try:
        _nat.layer_norm_backward(dy._core(), x._core(), mean._core(), rstd._core(), _core(weight), dx._core(), dw._core(),
                                 db._core(), q._stream)
    except (TypeError, ValueError):
        return None
    return dx, dw, db


def _direct_embedding(table, ids, scale, out):
    if type(table) is not usm_ndarray or type(ids) is not usm_ndarray or type(scale) is not float or len(table._shape) != 2:
        return None
    q = table._queue
    if not _plain(q, ids) or not _plain_rows(q, table, out) or ids._dtype not in _INDEX or table._dtype not in _ACCUMULATION:
        return None
    out = _new(ids._shape + table._shape[1:], table._dtype, q) if out is None else out
    try:
        _nat.embedding(table._core(), ids._core(), scale, out._core(), q._stream)
    except (TypeError, ValueError):
        return None
    return out


def _direct_distillation(logits, teacher_logits, teacher_index, temperature):
    """Whether the inputs of a distillation are ready for the library."""
    if type(logits) is not usm_ndarray or type(temperature) is not float:
        return False
    acc = _ACCUMULATION.get(logits._dtype)
    return (acc is not None and _plain_rows(logits._queue, logits) and _plain(logits._queue, teacher_logits, teacher_index)
            and teacher_logits is not None and teacher_index is not None and teacher_logits._dtype == acc
            and teacher_index._dtype in _INDEX and len(logits._shape) > 0
            and teacher_logits._shape[:-1] == logits._shape[:-1] and teacher_index._shape == teacher_logits._shape)


# ------------------------------------------------------------------------------------ layer normalisation
class _Normalized:
    """The axes of a layer normalisation: the kernel sees the remaining axes, then one axis with all of the
    normalised ones."""

    def __init__(self, x, axis):
        nd = len(x._shape)
        if nd == 0:
            raise ValueError("layer_norm needs an array of at least one dimension")
        axes = normalize_axis_tuple(axis if isinstance(axis, (tuple, list)) else (axis,), nd, "axis")
        if not axes:
            raise ValueError("layer_norm needs at least one axis")
        self.perm = [i for i in range(nd) if i not in axes] + list(axes)
        self.trailing = self.perm == list(range(nd))
        self.plain = self.trailing and len(axes) == 1
        self.inner = tuple(x._shape[a] for a in axes)
        self.outer = tuple(x._shape[i] for i in self.perm[:nd - len(axes)])
        self.n = 1
        for s in self.inner:
            self.n *= s
        if self.n == 0:
            raise ValueError("normalization cannot be performed over zero-size axes")
        self.shape = self.outer + (self.n,)
        self.full = x._shape

    def view(self, x):
        """`x` in the kernel's shape without a copy, or None."""
        if self.plain:
            return x
        try:
            return reshape(permute_dims(x, self.perm), self.shape, copy=False)
        except ValueError:
            return None

    def rows(self, x, q):
        v = self.view(x)
        if v is None:
            v = reshape(_dense(permute_dims(x, self.perm), q), self.shape)
        return _rows(v, q)

    def weight(self, w, q, what):
        if w is None:
            return None
        if w._shape != self.inner:
            raise ValueError(f"{what}: expected shape {self.inner}, got {w._shape}")
        w = _dense(w, q)
        return w if len(w._shape) == 1 else reshape(w, (self.n,))

    def stat(self, s, dt, q, what):
        if s._shape != self.outer:
            raise ValueError(f"{what}: expected shape {self.outer}, got {s._shape}")
        if s._dtype != dt:
            raise ValueError(f"{what}: type {dt} is needed, got {s._dtype}")
        return _dense(s, q)

    def back(self, y):
        """A result in the kernel's shape as the caller's."""
        if self.plain:
            return y
        inv = sorted(range(len(self.perm)), key=lambda d: self.perm[d])
        return permute_dims(reshape(y, self.outer + self.inner), inv)

    def out(self, target, dtype, q, inputs, in_place):
        """The result with the shape of x, and the array in the kernel's shape that stands for it."""
        o = _Out(target, self.full, dtype, q, inputs, in_place, walkable=self.plain, allocate=False)
        o.direct = o.direct and self.trailing
        if not o.direct:
            return o, _empty(self.shape, dtype, q)
        return o, target if self.plain else reshape(target, self.shape)

    def finish(self, o, kernel_out, q):
        if o.direct:
            return o.target
        o.buf = self.back(kernel_out)
        return o.finish(q)


def _check_weights(x, *weights):
    types = {w._dtype for w in weights if w is not None}
    if len(types) > 1:
        raise ValueError("weight and bias must have the same type")
    for dt in types:
        if dt != x._dtype and not (x._dtype == _HALF and dt == _SINGLE):
            raise TypeError(f"weight: type {dt} does not go with {x._dtype} data")
    return types.pop() if types else x._dtype


def layer_norm(x, weight=None, bias=None, /, *, axis=-1, eps=1e-5, return_stats=False, out=None):
    """Layer normalisation: ``(x - mean) * rstd * weight + bias`` with the mean and
    ``rstd = 1 / sqrt(var + eps)`` taken over `axis`.

    x : float16, float32 or float64 array.
    weight, bias : arrays of the shape of the normalised axes (in the order of `axis`), both of the type of
        `x` or, for float16 data, both float32; either may be None.
    axis : int or tuple of ints.
    return_stats : also return ``mean`` and ``rstd`` (shape of the remaining axes, float32, or float64 for
        float64 data), which :func:`layer_norm_backward` takes.
    out : array for the result, or with `return_stats` a tuple of three (None: allocated).  The result may
        be written over `x`.
    """
    if axis == -1 and _nat is not None:
        res = _direct_layer_norm(x, weight, bias, eps, return_stats, out)
        if res is not None:
            return res
    _check_array(x, "x")
    for w, what in ((weight, "weight"), (bias, "bias")):
        if w is not None:
            _check_array(w, what)
    acc = _accumulation_type(x, "x")
    eps = _number(eps, "eps")
    if not 0 <= eps < float("inf"):
        raise ValueError("eps must be a finite number that is not negative")
    q = _execution_queue(x, weight, bias)
    _check_weights(x, weight, bias)
    axes = _Normalized(x, axis)
    if return_stats:
        out = _unpack_out(out, 3, "layer_norm")
    else:
        if out is not None and not isinstance(out, usm_ndarray):
            raise TypeError(f"output array must be of usm_ndarray type, got {type(out)}")
        out = (out, None, None)
    inputs = (x, weight, bias)
    w, b = axes.weight(weight, q, "weight"), axes.weight(bias, q, "bias")
    y, y_rows = axes.out(out[0], x._dtype, q, inputs, (x,))
    stats = [_Out(o, axes.outer, acc, q, inputs) for o in out[1:]] if return_stats else []
    tri._layer_norm(axes.rows(x, q), w, b, eps, y_rows, *([s.buf for s in stats] or (None, None)), sycl_queue=q)
    res = axes.finish(y, y_rows, q)
    return (res, *[s.finish(q) for s in stats]) if return_stats else res


def layer_norm_backward(dy, x, mean, rstd, weight=None, /, *, axis=-1, weight_grads=True, out=None):
    """Gradients of :func:`layer_norm`: ``(dx, dweight, dbias)``.

    dy : gradient of the result, of the shape and type of `x`.
    mean, rstd : the statistics that ``layer_norm(..., return_stats=True)`` returned for `x`.
    weight : the weight of the forward call, or None (a weight of ones).
    weight_grads : False leaves the last two gradients out: ``(dx, None, None)``.
    out : tuple of three arrays or None.  dweight and dbias have the type of `weight` (of `x` without one);
        without a weight, float32 arrays in `out` are accepted for float16 data.  dx may be written over `dy`
        or `x`.

    The sums over the rows have a fixed order: the same call gives the same bits.
    """
    if axis == -1 and _nat is not None:
        res = _direct_layer_norm_backward(dy, x, mean, rstd, weight, weight_grads, out)
        if res is not None:
            return res
    for a, what in ((dy, "dy"), (x, "x"), (mean, "mean"), (rstd, "rstd")):
        _check_array(a, what)
    if weight is not None:
        _check_array(weight, "weight")
    acc = _accumulation_type(x, "x")
    if dy._shape != x._shape:
        raise ValueError(f"dy: expected shape {x._shape}, got {dy._shape}")
    if dy._dtype != x._dtype:
        raise ValueError(f"dy: type {x._dtype} is needed, got {dy._dtype}")
    q = _execution_queue(dy, x, mean, rstd, weight)
    out = _unpack_out(out, 3, "layer_norm_backward")
    if not weight_grads and (out[1] is not None or out[2] is not None):
        raise ValueError("`out` has arrays for gradients that weight_grads=False leaves out")
    given = next((o._dtype for o in out[1:] if o is not None), None)
    wt = _check_weights(x, weight)
    if weight is None and given is not None and x._dtype == _HALF and given == _SINGLE:
        wt = _SINGLE
    axes = _Normalized(x, axis)
    inputs = (dy, x, mean, rstd, weight)
    w, m, r = axes.weight(weight, q, "weight"), axes.stat(mean, acc, q, "mean"), axes.stat(rstd, acc, q, "rstd")
    dx, dx_rows = axes.out(out[0], x._dtype, q, inputs, (dy, x))
    grads = []
    if weight_grads:
        for o in out[1:]:
            if o is not None and o._shape != axes.inner:
                raise ValueError("The shape of input and output arrays are inconsistent. "
                                 f"Expected output shape is {axes.inner}, got {o._shape}")
            grads.append(_Out(o, axes.inner, wt, q, inputs))
    flat = [reshape(g.buf, (axes.n,)) for g in grads] or [None, None]
    tri._layer_norm_backward(axes.rows(dy, q), axes.rows(x, q), m, r, w, dx_rows, *flat, sycl_queue=q)
    res = axes.finish(dx, dx_rows, q)
    return (res, *([g.finish(q) for g in grads] or (None, None)))


# ---------------------------------------------------------------------------------------------- embedding
def _check_ids(ids):
    _check_array(ids, "ids")
    if ids._dtype.kind not in "iu":
        raise TypeError(f"ids: an integer array is needed, got {ids._dtype}")


def _ids(ids, q):
    return _typed(ids, ids._dtype if ids._dtype in _INDEX else np.dtype("i8"), q)


def embedding(table, ids, /, *, scale=1.0, out=None):
    """Rows of `table` by number: ``out[..., :] = scale * table[ids[...], :]``.

    table : two-dimensional float16, float32 or float64 array.
    ids : integer array of any shape.  An id outside ``[0, len(table))``, such as the -1 of a padded batch,
        names no row: its result is a row of zeros.  (uint64 ids of 2**63 and above are outside, too.)
    out : array of shape ``ids.shape + table.shape[1:]`` and the type of `table`.
    """
    if _nat is not None:
        res = _direct_embedding(table, ids, scale, out)
        if res is not None:
            return res
    _check_array(table, "table")
    _check_ids(ids)
    _accumulation_type(table, "table")
    scale = _number(scale, "scale")
    if len(table._shape) != 2:
        raise ValueError(f"table: a two-dimensional array is needed, got {len(table._shape)} dimensions")
    q = _execution_queue(table, ids)
    if out is not None:
        _check_array(out, "out")
    o = _Out(out, ids._shape + table._shape[1:], table._dtype, q, (table, ids), walkable=True)
    t = table if table._shape[1] <= 1 or table._strides[1] == 1 else _dense(table, q)
    tri._embedding(t, _ids(ids, q), scale, o.buf, sycl_queue=q)
    return o.finish(q)


def embedding_backward(dout, ids, num_rows, /, *, scale=1.0, dtype=None, out=None):
    """Gradient of :func:`embedding` with respect to its table, of shape ``(num_rows, dout.shape[-1])``:
    row v is ``scale`` times the sum of ``dout[i]`` over the places where ``ids[i] == v``, zeros where there
    are none.  Ids outside ``[0, num_rows)`` add nothing.

    dout : float16, float32 or float64 array of shape ``ids.shape + (n,)``.
    dtype : type of the result: that of `dout` (default, or that of `out`), or float32 for float16 data.
    out : array for the result; it is overwritten, not added to.

    Sums are float32 (float64 for float64 data) in a fixed order: the same call gives the same bits.
    """
    _check_array(dout, "dout")
    _check_ids(ids)
    _accumulation_type(dout, "dout")
    scale = _number(scale, "scale")
    if isinstance(num_rows, (bool, np.bool_)) or not isinstance(num_rows, (int, np.integer)):
        raise TypeError(f"num_rows: an integer is needed, got {type(num_rows)}")
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    if dout._shape[:-1] != ids._shape or len(dout._shape) != len(ids._shape) + 1:
        raise ValueError(f"dout: expected shape {ids._shape} and one further axis, got {dout._shape}")
    q = _execution_queue(dout, ids)
    if out is not None:
        _check_array(out, "out")
    dt = np.dtype(dtype) if dtype is not None else out._dtype if out is not None else dout._dtype
    if dt != dout._dtype and not (dout._dtype == _HALF and dt == _SINGLE):
        raise TypeError(f"dtype: a gradient of type {dt} does not go with {dout._dtype} data")
    o = _Out(out, (int(num_rows), dout._shape[-1]), dt, q, (dout, ids), walkable=True)
    tri._embedding_backward(_rows(dout, q), _ids(ids, q), scale, o.buf, sycl_queue=q)
    return o.finish(q)


# ------------------------------------------------------------------------------------------- distillation
def _distillation_args(logits, teacher_logits, teacher_index, temperature):
    _check_array(logits, "logits")
    _check_array(teacher_logits, "teacher_logits")
    _check_array(teacher_index, "teacher_index")
    acc = _accumulation_type(logits, "logits")
    _accumulation_type(teacher_logits, "teacher_logits")
    temperature = _number(temperature, "temperature")
    if len(logits._shape) == 0:
        raise ValueError("logits: an array of at least one dimension is needed")
    if teacher_index._dtype.kind not in "iu":
        raise TypeError(f"teacher_index: an integer array is needed, got {teacher_index._dtype}")
    if teacher_logits._shape[:-1] != logits._shape[:-1] or len(teacher_logits._shape) != len(logits._shape):
        raise ValueError(f"teacher_logits: expected shape {logits._shape[:-1]} and one further axis, "
                         f"got {teacher_logits._shape}")
    if teacher_index._shape != teacher_logits._shape:
        raise ValueError(f"teacher_index: expected shape {teacher_logits._shape}, got {teacher_index._shape}")
    return acc, temperature


def _distillation_inputs(logits, teacher_logits, teacher_index, acc, q):
    index_type = teacher_index._dtype if teacher_index._dtype in _INDEX else np.dtype("i8")
    return _rows(logits, q), _typed(teacher_logits, acc, q), _typed(teacher_index, index_type, q)


def _row_gradient(dloss, shape, acc, q):
    """`dloss` as an array of one value a row, or of no dimensions, in the accumulation type."""
    if isinstance(dloss, usm_ndarray):
        if dloss._shape not in ((), shape):
            raise ValueError(f"dloss: expected shape {shape} or (), got {dloss._shape}")
        _accumulation_type(dloss, "dloss")
        return _typed(dloss, acc, q)
    value = _number(dloss, "dloss")
    res = _empty((), acc, q)
    ti._full_usm_ndarray(value, res, q)
    return res


def distillation_loss(logits, teacher_logits, teacher_index, /, *, temperature=1.0, return_stats=False, out=None):
    """Divergence of a student's distribution from a teacher's, known by its top logits, for every row:
    ``T**2 * sum(p * (log p - log q))`` with ``p = softmax(teacher_logits / T)`` over the row's K entries
    and ``q = softmax(logits / T)`` over all V columns, taken at the entries' columns.

    logits : array (..., V) of float16, float32 or float64.
    teacher_logits : floating array (..., K), K at most 1024.
    teacher_index : integer array (..., K): the columns of the entries.  An entry whose column lies outside
        ``[0, V)`` (the -1 of a shorter list) or whose logit is -inf does not count; a row without entries
        (padding, a prompt) has loss 0.  A column named twice counts twice.
    temperature : T, a positive number.
    return_stats : also return what :func:`distillation_loss_backward` takes, (..., 2): the row's largest
        logit, and log of the sum of ``exp((logits - largest) / T)``; zeros for a row without entries.
    out : array for the losses, or with `return_stats` a tuple of two (None: allocated).

    Loss and statistics are float32, or float64 for float64 logits.  Where q is 0 and p is not (a student
    logit of -inf at the teacher's column) the loss is +inf; NaN and +inf in a row that counts make its loss and
    its gradient NaN.
    """
    if _nat is not None and _direct_distillation(logits, teacher_logits, teacher_index, temperature):
        outs, q = _outs(out, 2 if return_stats else 1), logits._queue
        if outs is not None and _plain(q, *outs):
            acc, lead = teacher_logits._dtype, logits._shape[:-1]
            loss = _new(lead, acc, q) if outs[0] is None else outs[0]
            stats = None if not return_stats else _new(lead + (2,), acc, q) if outs[1] is None else outs[1]
            try:
                _nat.distillation_loss(logits._core(), teacher_logits._core(), teacher_index._core(), temperature,
                                       loss._core(), _core(stats), q._stream)
                return (loss, stats) if return_stats else loss
            except (TypeError, ValueError):
                pass
    acc, temperature = _distillation_args(logits, teacher_logits, teacher_index, temperature)
    q = _execution_queue(logits, teacher_logits, teacher_index)
    if return_stats:
        out = _unpack_out(out, 2, "distillation_loss")
    else:
        if out is not None:
            _check_array(out, "out")
        out = (out,)
    inputs = (logits, teacher_logits, teacher_index)
    lead = logits._shape[:-1]
    loss = _Out(out[0], lead, acc, q, inputs)
    stats = _Out(out[1], lead + (2,), acc, q, inputs) if return_stats else None
    tri._distillation_loss(*_distillation_inputs(*inputs, acc, q), temperature, loss.buf,
                           stats.buf if return_stats else None, sycl_queue=q)
    return (loss.finish(q), stats.finish(q)) if return_stats else loss.finish(q)


def distillation_loss_backward(dloss, logits, teacher_logits, teacher_index, stats, /, *, temperature=1.0, out=None):
    """Gradient of :func:`distillation_loss` with respect to `logits`:
    ``dloss * T * (q - p)``, zeros in rows without entries; q is 0 where a logit is -inf.

    dloss : gradient of the losses: one value a row, or one (an array without dimensions or a number) for all.
    stats : the statistics that ``distillation_loss(..., return_stats=True)`` returned for these logits.
    out : array of the shape and type of `logits`; the result may be written over `logits`.
    """
    if _nat is not None and _direct_distillation(logits, teacher_logits, teacher_index, temperature):
        q = logits._queue
        if type(dloss) is usm_ndarray and stats is not None and _plain(q, dloss, stats) and _plain_rows(q, out):
            dz = _new(logits._shape, logits._dtype, q) if out is None else out
            try:
                _nat.distillation_loss_backward(dloss._core(), logits._core(), teacher_logits._core(), teacher_index._core(),
                                                stats._core(), temperature, dz._core(), q._stream)
                return dz
            except (TypeError, ValueError):
                pass
    acc, temperature = _distillation_args(logits, teacher_logits, teacher_index, temperature)
    _check_array(stats, "stats")
    lead = logits._shape[:-1]
    if stats._shape != lead + (2,):
        raise ValueError(f"stats: expected shape {lead + (2,)}, got {stats._shape}")
    if stats._dtype != acc:
        raise ValueError(f"stats: type {acc} is needed, got {stats._dtype}")
    given = dloss if isinstance(dloss, usm_ndarray) else None
    q = _execution_queue(logits, teacher_logits, teacher_index, stats, given)
    if out is not None:
        _check_array(out, "out")
    g = _row_gradient(dloss, lead, acc, q)
    dz = _Out(out, logits._shape, logits._dtype, q, (logits, teacher_logits, teacher_index, stats, given), (logits,),
              walkable=True)
    z, top, index = _distillation_inputs(logits, teacher_logits, teacher_index, acc, q)
    tri._distillation_loss_backward(g, z, top, index, _dense(stats, q), temperature, dz.buf, sycl_queue=q)
    return dz.finish(q)


def distillation_loss_and_grad(logits, teacher_logits, teacher_index, dloss=1.0, /, *, temperature=1.0, out=None):
    """Losses and the gradient with respect to `logits` in one call: what :func:`distillation_loss` and
    :func:`distillation_loss_backward` return, for a `dloss` that is known beforehand (a weight per row, or
    ``1 / rows`` for the mean over the rows).

    out : tuple of two arrays (None: allocated); the gradient may be written over `logits`.
    """
    if _nat is not None and _direct_distillation(logits, teacher_logits, teacher_index, temperature):
        outs, q = _outs(out, 2), logits._queue
        if outs is not None and type(dloss) is usm_ndarray and _plain(q, dloss, outs[0]) and _plain_rows(q, outs[1]):
            loss = _new(logits._shape[:-1], teacher_logits._dtype, q) if outs[0] is None else outs[0]
            dz = _new(logits._shape, logits._dtype, q) if outs[1] is None else outs[1]
            try:
                _nat.distillation_loss_and_grad(logits._core(), teacher_logits._core(), teacher_index._core(), dloss._core(),
                                                temperature, loss._core(), dz._core(), q._stream)
                return loss, dz
            except (TypeError, ValueError):
                pass
    acc, temperature = _distillation_args(logits, teacher_logits, teacher_index, temperature)
    lead = logits._shape[:-1]
    given = dloss if isinstance(dloss, usm_ndarray) else None
    q = _execution_queue(logits, teacher_logits, teacher_index, given)
    out = _unpack_out(out, 2, "distillation_loss_and_grad")
    g = _row_gradient(dloss, lead, acc, q)
    inputs = (logits, teacher_logits, teacher_index, given)
    loss = _Out(out[0], lead, acc, q, inputs)
    dz = _Out(out[1], logits._shape, logits._dtype, q, inputs, (logits,), walkable=True)
    z, top, index = _distillation_inputs(*inputs[:3], acc, q)
    tri._distillation_loss_and_grad(z, top, index, g, temperature, loss.buf, dz.buf, sycl_queue=q)
    return loss.finish(q), dz.finish(q)
