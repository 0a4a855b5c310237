"""Python face of the row operators of the C ABI (layer normalisation, embedding lookup, distillation loss
and their gradients): ``_<operator>(arrays..., sycl_queue)``, in the manner of the reference's native
modules (dpnp/tensor/libtensor/source/tensor_reductions.cpp:40-43).  Optional arrays are ``None``."""

from __future__ import annotations

import ctypes as C

from .. import _lib
from .._lib import check, lib
from ._tensor_impl import _check_queue, _events, _stream

_nat = _lib.native


def _make(name):
    native_fn = getattr(_nat, name, None) if _nat is not None else None
    c_fn = getattr(lib, f"dpb_{name}")

    def call(*args, sycl_queue, depends=()):
        """`args` in the order of the C entry point: arrays, None for absent ones, and numbers."""
        arrays = [a for a in args if a is not None and type(a) is not float]
        _check_queue(sycl_queue, *arrays)
        if native_fn is not None:
            native_fn(*[a if a is None or type(a) is float else a._core() for a in args], sycl_queue._stream)
            return _events(sycl_queue)
        descriptors = [a if a is None or type(a) is float else a._descriptor() for a in args]
        check(c_fn(*[C.byref(d[0]) if type(d) is tuple else d for d in descriptors], _stream(sycl_queue)))
        return _events(sycl_queue)

    call.__name__ = f"_{name}"
    return call


_layer_norm = _make("layer_norm")
_layer_norm_backward = _make("layer_norm_backward")
_embedding = _make("embedding")
_embedding_backward = _make("embedding_backward")
_distillation_loss = _make("distillation_loss")
_distillation_loss_backward = _make("distillation_loss_backward")
_distillation_loss_and_grad = _make("distillation_loss_and_grad")
