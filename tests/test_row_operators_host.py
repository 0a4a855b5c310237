"""Refusals and layout decisions of the row operators (layer normalisation, embedding lookup, distillation loss),
on the CPU: arrays are views over a stand-in memory object, nothing is launched."""

import ctypes as C
import math

import numpy as np
import pytest

import dpnp_b200 as dp
from dpnp_b200 import _lib, memory
from dpnp_b200.tensor import _row_functions as rf
from dpnp_b200.tensor._usmarray import _dense_strides, usm_ndarray

NAN = float("nan")


class _Mem:
    nbytes = 1 << 50
    ptr = _ptr = 4096


_at = [1 << 20]


def arr(shape, dt="f4", strides=None, at=None, queue=7, writable=True, device=0):
    if at is None:
        _at[0] += 1 << 30
        at = _at[0]
    shape = tuple(shape)
    q = memory.StreamQueue(device, stream=queue)
    return usm_ndarray._view(_Mem, at, shape, tuple(strides if strides is not None else _dense_strides(shape)),
                             np.dtype(dt), q, writable)


def c_call(name, *args):
    """The C entry point on descriptors; the status code."""
    keep = [a if a is None or isinstance(a, float) else a._descriptor() for a in args]
    fn = getattr(_lib.lib, f"dpb_{name}")
    return fn(*[C.byref(a[0]) if isinstance(a, tuple) else a for a in keep], None)


X = lambda *s, **k: arr(s or (4, 8), **k)  # noqa: E731


# ----------------------------------------------------------------------------------- Python layer refusals
@pytest.mark.parametrize("call,error", [
    (lambda: dp.layer_norm(np.ones((2, 2))), TypeError),
    (lambda: dp.layer_norm(X(dt="i4")), TypeError),
    (lambda: dp.layer_norm(X(dt="c8")), TypeError),
    (lambda: dp.layer_norm(X(), X(8, dt="f8")), TypeError),
    (lambda: dp.layer_norm(X(), X(8, dt="f2")), TypeError),
    (lambda: dp.layer_norm(X(dt="f2"), X(8, dt="f2"), X(8, dt="f4")), ValueError),
    (lambda: dp.layer_norm(X(), X(7)), ValueError),
    (lambda: dp.layer_norm(X(), X(1, 8)), ValueError),
    (lambda: dp.layer_norm(X(), None, X(4), axis=-1), ValueError),
    (lambda: dp.layer_norm(X(), axis=2), (ValueError, IndexError)),
    (lambda: dp.layer_norm(X(), axis=(0, 0)), ValueError),
    (lambda: dp.layer_norm(X(), axis=()), ValueError),
    (lambda: dp.layer_norm(arr(())), ValueError),
    (lambda: dp.layer_norm(arr((3, 0))), ValueError),
    (lambda: dp.layer_norm(X(), eps=-1e-5), ValueError),
    (lambda: dp.layer_norm(X(), eps=NAN), ValueError),
    (lambda: dp.layer_norm(X(), eps=math.inf), ValueError),
    (lambda: dp.layer_norm(X(), eps="1"), TypeError),
    (lambda: dp.layer_norm(X(), eps=True), TypeError),
    (lambda: dp.layer_norm(X(), arr((8,), queue=8)), memory.ExecutionPlacementError),
    (lambda: dp.layer_norm(X(), out=arr((4, 8), queue=8)), memory.ExecutionPlacementError),
    (lambda: dp.layer_norm(X(), out=arr((4, 8), writable=False)), ValueError),
    (lambda: dp.layer_norm(X(), out=arr((8, 4))), ValueError),
    (lambda: dp.layer_norm(X(), out=arr((4, 8), "f8")), ValueError),
    (lambda: dp.layer_norm(X(), out=arr((4, 8), strides=(0, 1))), ValueError),
    (lambda: dp.layer_norm(X(), return_stats=True, out=X()), TypeError),
    (lambda: dp.layer_norm(X(), return_stats=True, out=(X(), None)), TypeError),
    (lambda: dp.layer_norm(X(), return_stats=True, out=(None, arr((4,), at=4096), arr((4,), at=4096))), ValueError),
    (lambda: dp.layer_norm_backward(X(4, 9), X(), X(4), X(4)), ValueError),
    (lambda: dp.layer_norm_backward(X(dt="f8"), X(), X(4), X(4)), ValueError),
    (lambda: dp.layer_norm_backward(X(), X(), X(4), X(4), weight_grads=False, out=(None, X(8), None)), ValueError),
    (lambda: dp.embedding(X(8), X(3, dt="i4")), ValueError),
    (lambda: dp.embedding(X(dt="i4"), X(3, dt="i4")), TypeError),
    (lambda: dp.embedding(X(), X(3)), TypeError),
    (lambda: dp.embedding(X(), X(3, dt="?")), TypeError),
    (lambda: dp.embedding(X(), X(3, dt="i4"), scale=1j), TypeError),
    (lambda: dp.embedding(X(), X(3, dt="i4"), out=X(3, 7)), ValueError),
    (lambda: dp.embedding(X(), arr((3,), "i4", queue=9)), memory.ExecutionPlacementError),
    (lambda: dp.embedding_backward(X(3, 8), X(4, dt="i4"), 10), ValueError),
    (lambda: dp.embedding_backward(X(3, 8), X(3, dt="i4"), -1), ValueError),
    (lambda: dp.embedding_backward(X(3, 8), X(3, dt="i4"), 10.0), TypeError),
    (lambda: dp.embedding_backward(X(3, 8), X(3, dt="i4"), 10, dtype="f2"), TypeError),
    (lambda: dp.embedding_backward(X(3, 8), X(3, dt="i4"), 10, out=X(10, 8, dt="f8")), TypeError),
    (lambda: dp.distillation_loss(X(4, 50, dt="i4"), X(4, 3), X(4, 3, dt="i4")), TypeError),
    (lambda: dp.distillation_loss(X(4, 50), X(5, 3), X(5, 3, dt="i4")), ValueError),
    (lambda: dp.distillation_loss(X(4, 50), X(4, 3), X(4, 2, dt="i4")), ValueError),
    (lambda: dp.distillation_loss(X(4, 50), X(4, 3), X(4, 3)), TypeError),
    (lambda: dp.distillation_loss(X(4, 50), X(4, 3, dt="i4"), X(4, 3, dt="i4")), TypeError),
    (lambda: dp.distillation_loss(X(4, 50), X(3), X(3, dt="i4")), ValueError),
    (lambda: dp.distillation_loss(arr(()), arr(()), arr((), "i4")), ValueError),
    (lambda: dp.distillation_loss(X(4, 50), X(4, 3), X(4, 3, dt="i4"), temperature="1"), TypeError),
    (lambda: dp.distillation_loss(X(4, 50), X(4, 3), X(4, 3, dt="i4"), return_stats=True, out=X(4)), TypeError),
    (lambda: dp.distillation_loss_backward(X(4), X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4, 3)), ValueError),
    (lambda: dp.distillation_loss_backward(X(4), X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4, 2, dt="f8")), ValueError),
    (lambda: dp.distillation_loss_backward(X(5), X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4, 2), out=X(4, 50)), ValueError),
    (lambda: dp.distillation_loss_and_grad(X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4, 1)), ValueError),
    (lambda: dp.distillation_loss_and_grad(X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4), out=(X(4), X(4, 49))), ValueError),
])
def test_arguments_are_refused_before_anything_is_allocated(call, error):
    with pytest.raises(error):
        call()


# --------------------------------------------------------------------------------------- C layer refusals
def _norm(x=None, w=None, b=None, eps=1e-5, y=None, mean=None, rstd=None):
    x = X() if x is None else x
    return c_call("layer_norm", x, w, b, eps, arr(x.shape, x.dtype) if y is None else y, mean, rstd)


def _distil(z=None, t=None, j=None, temp=1.0, loss=None, stats=None):
    z, t, j, loss = (d if a is None else a for a, d in ((z, X(4, 50)), (t, X(4, 3)), (j, X(4, 3, dt="i4")), (loss, X(4))))
    return c_call("distillation_loss", z, t, j, temp, loss, stats)


@pytest.mark.parametrize("call", [
    lambda: _norm(arr((4, 8), strides=(1, 4))),                                # not unit-stride rows
    lambda: _norm(arr((4, 4, 4, 8), strides=(9999, 512, 40, 1))),              # three levels of rows
    lambda: _norm(arr((4, 8), at=4098)),                                       # misaligned elements
    lambda: _norm(eps=-1.0),
    lambda: _norm(eps=NAN),
    lambda: _norm(w=arr((8,), strides=(2,))),
    lambda: _norm(w=X(8), b=X(8, dt="f8")),
    lambda: _norm(w=X(8, dt="f8")),
    lambda: _norm(y=X(4, 8, writable=False)),
    lambda: _norm(y=arr((4, 8), strides=(4, 1))),                              # rows overlap one another
    lambda: _norm(x=arr((4, 8), at=4096), y=arr((4, 8), at=4100)),             # partial overlap
    lambda: _norm(x=arr((4, 8), at=4096), mean=arr((4,), at=4096)),
    lambda: _norm(mean=arr((4,), at=4096), rstd=arr((4,), at=4096)),
    lambda: _norm(mean=arr((4,), strides=(2,))),
    lambda: _norm(mean=X(4, dt="f8")),
    lambda: _norm(y=X(4, 8, device=1)),
    lambda: _norm(arr((1 << 31, 1), "f2"), y=arr((1 << 31, 1), "f2")),
    lambda: c_call("layer_norm", None, None, None, 1e-5, X(), None, None),
    lambda: c_call("layer_norm_backward", X(), X(), None, X(4), None, X(), None, None),
    lambda: c_call("layer_norm_backward", X(), X(), X(4), X(4), None, X(), X(8), None),
    lambda: c_call("layer_norm_backward", arr((4, 8), at=4096), X(), X(4), X(4), None, X(), arr((8,), at=4096), X(8)),
    lambda: c_call("embedding", X(), X(3, dt="i2"), 1.0, X(3, 8)),
    lambda: c_call("embedding", X(), arr((3,), "i4", strides=(2,)), 1.0, X(3, 8)),
    lambda: c_call("embedding", arr((4, 8), strides=(1, 4)), X(3, dt="i4"), 1.0, X(3, 8)),
    lambda: c_call("embedding", arr((4, 8), at=4096), X(3, dt="i4"), 1.0, arr((3, 8), at=4096)),
    lambda: c_call("embedding", X(), X(3, dt="i4"), 1.0, X(3, 8, dt="f8")),
    lambda: c_call("embedding_backward", X(3, 8), X(3, dt="i4"), 1.0, X(5, 8, dt="f2")),
    lambda: c_call("embedding_backward", X(3, 8), X(3, dt="i4"), 1.0, arr((5, 8), strides=(0, 1))),
    lambda: c_call("embedding_backward", X(3, 8), X(4, dt="i4"), 1.0, X(5, 8)),
    lambda: _distil(temp=0.0),
    lambda: _distil(temp=-1.0),
    lambda: _distil(temp=NAN),
    lambda: _distil(temp=math.inf),
    lambda: _distil(temp=1e-30),                                               # T^2 vanishes in float32
    lambda: _distil(temp=1e30),
    lambda: _distil(X(4, 0)),
    lambda: _distil(t=X(4, 1025), j=X(4, 1025, dt="i4")),
    lambda: _distil(t=X(4, 3, dt="f8")),
    lambda: _distil(j=X(4, 3, dt="u4")),
    lambda: _distil(loss=arr((4,), strides=(2,))),
    lambda: _distil(stats=X(4, 3)),
    lambda: _distil(z=arr((4, 50), at=4096), loss=arr((4,), at=4096)),
    lambda: c_call("distillation_loss_and_grad", X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4), 1.0, X(4), None),
    lambda: c_call("distillation_loss_and_grad", X(4, 50), X(4, 3), X(4, 3, dt="i4"), X(4), 1.0,
                   arr((4,), at=4096), arr((4, 50), at=4096)),
    lambda: c_call("distillation_loss_backward", X(4), X(4, 50), X(4, 3), X(4, 3, dt="i4"), None, 1.0, X(4, 50)),
    lambda: c_call("distillation_loss_backward", X(4), arr((4, 50), at=4096), X(4, 3), X(4, 3, dt="i4"), X(4, 2), 1.0,
                   arr((4, 50), at=4100)),
])
def test_the_c_entry_points_refuse_what_the_kernels_cannot_take(call):
    assert call() in (_lib.ERR_VALUE, _lib.ERR_TYPE)
    assert _lib.last_error()


def test_empty_calls_succeed_without_a_launch():
    before = _lib.launch_count()
    assert _norm(X(0, 8)) == _lib.OK
    assert c_call("embedding", X(), X(0, dt="i4"), 1.0, X(0, 8)) == _lib.OK
    assert c_call("embedding_backward", X(3, 8), X(3, dt="i4"), 1.0, X(0, 8)) == _lib.OK
    assert _distil(X(0, 50), X(0, 3), X(0, 3, dt="i4"), loss=X(0)) == _lib.OK
    assert _lib.launch_count() == before


# ------------------------------------------------------------------------------------------------ layouts
@pytest.mark.parametrize("shape,strides,walks", [
    ((4, 8), (8, 1), True), ((4, 8), (11, 1), True), ((4, 8), (-8, 1), True), ((4, 8), (0, 1), True),
    ((4, 8), (8, 2), False), ((4, 8), (1, 4), False), ((2, 3, 8), (100, 8, 1), True), ((2, 3, 4, 8), (96, 32, 8, 1), True),
    ((2, 3, 4, 8), (500, 100, 8, 1), False), ((2, 1, 4, 8), (500, 77, 8, 1), True), ((4, 1), (5, 9), True), ((8,), (1,), True),
    ((), (), False), ((2, 3, 4, 8), (100, 32, 8, 1), True), ((2, 3, 4, 8), (96, 32, 10, 1), True),
])
def test_which_rows_are_walked_without_a_copy(shape, strides, walks):
    assert rf._walkable(shape, strides) is walks
    # the library draws the same line: it gets past the rows to the next check, the overlap of x and y
    if shape:
        same = _norm(arr(shape, strides=strides, at=4096), y=arr(shape, at=4096 + 4))
        assert same == _lib.ERR_VALUE and ("overlapping" in _lib.last_error()) is walks


@pytest.mark.parametrize("axis,shape", [(-1, (5, 6, 7)), (1, (5, 6, 7)), ((1, 2), (5, 6, 7)), ((2, 0), (5, 6, 7)), (0, (9,))])
def test_normalised_axes_are_moved_to_the_end(axis, shape):
    x = arr(shape)
    a = rf._Normalized(x, axis)
    axes = tuple(i % len(shape) for i in (axis if isinstance(axis, tuple) else (axis,)))
    rest = tuple(s for i, s in enumerate(shape) if i not in axes)
    assert a.inner == tuple(shape[i] for i in axes) and a.outer == rest
    assert a.shape == rest + (math.prod(a.inner),)
    assert a.back(arr(a.shape)).shape == shape


def test_the_functions_are_public_in_both_layers():
    import dpnp_b200.tensor as dpt

    for name in ("layer_norm", "layer_norm_backward", "embedding", "embedding_backward", "distillation_loss",
                 "distillation_loss_backward", "distillation_loss_and_grad"):
        assert getattr(dp, name).__doc__ == getattr(dpt, name).__doc__ and getattr(dp, name).__doc__


def _one_queue():
    """Valid positional arguments of every operator, all on one queue object (the direct route)."""
    q = memory.StreamQueue(0, stream=7)

    def a(*shape, dt="f4"):
        _at[0] += 1 << 30
        return usm_ndarray._view(_Mem, _at[0], shape, tuple(_dense_strides(shape)), np.dtype(dt), q, True)

    z, t, j = a(4, 50), a(4, 3), a(4, 3, dt="i4")
    return {"layer_norm": [a(4, 8)], "layer_norm_backward": [a(4, 8), a(4, 8), a(4), a(4)], "embedding": [a(4, 8), a(3, dt="i4")],
            "embedding_backward": [a(3, 8), a(3, dt="i4"), 10], "distillation_loss": [z, t, j],
            "distillation_loss_backward": [a(4), z, t, j, a(4, 2)], "distillation_loss_and_grad": [z, t, j, a(4)]}


@pytest.mark.parametrize("name", sorted(_one_queue()))
@pytest.mark.parametrize("layer", [dp, dp.tensor])
def test_a_required_argument_that_is_no_array_is_a_type_error(layer, name):
    args = _one_queue()[name]
    for i in range(len(args)):
        for wrong in (None, "1", [1.0], np.ones((4, 8), "f4"), 1j):
            with pytest.raises(TypeError):
                getattr(layer, name)(*args[:i], wrong, *args[i + 1:])
