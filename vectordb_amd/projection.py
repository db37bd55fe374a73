"""Learned maps of embeddings into a table's space: what Engine.project_* , insert_projected_dev and
search_projected_dev take (vdb_projection of include/vdb.h).

The weights stay the caller's tensors on the engine's GPU; a Projection holds references to them and their addresses.
Values that are changed in place are seen by the next call.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import VdbError

_DTYPES = {"torch.float32": _lib.F32, "torch.bfloat16": _lib.BF16, "torch.float16": _lib.F16}


def _dtype(t) -> int:
    """VDB_* number of a torch dtype, or of an engine dtype number."""
    if isinstance(t, int):
        if t not in (_lib.F32, _lib.BF16, _lib.F16):
            raise VdbError(_lib.EINVAL, "unknown dtype %r" % (t,))
        return t
    try:
        return _DTYPES[str(t)]
    except KeyError:
        raise VdbError(_lib.EINVAL, "dtype %s is not one of float32, bfloat16, float16" % (t,)) from None


def _check(name: str, t, shape, dtype: int) -> None:
    if tuple(t.shape) != tuple(shape):
        raise VdbError(_lib.EINVAL, "%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    if _dtype(t.dtype) != dtype:
        raise VdbError(_lib.EINVAL, "%s is %s" % (name, t.dtype))
    if not t.is_contiguous():
        raise VdbError(_lib.EINVAL, "%s is not contiguous" % name)


class Projection:
    """w [groups, dim_out, dim_in] (or [dim_out, dim_in]); adapters: a [adapters, rank, dim_in], b [adapters, dim_out, rank],
    scale [adapters] fp32 (1 if left out).  Tensors on one GPU; out_dtype: type of what calls write, the weights' own if left out."""

    def __init__(self, w, a=None, b=None, scale=None, out_dtype=None):
        if len(w.shape) == 2:
            w = w.reshape((1,) + tuple(w.shape))
        if len(w.shape) != 3:
            raise VdbError(_lib.EINVAL, "w must be [groups, dim_out, dim_in]")
        groups, dim_out, dim_in = (int(v) for v in w.shape)
        dtype = _dtype(w.dtype)
        _check("w", w, (groups, dim_out, dim_in), dtype)
        adapters = rank = 0
        if (a is None) != (b is None):
            raise VdbError(_lib.EINVAL, "an adapter needs both a and b")
        if a is None and scale is not None:
            raise VdbError(_lib.EINVAL, "scale without adapters")
        if a is not None:
            if len(a.shape) != 3:
                raise VdbError(_lib.EINVAL, "a must be [adapters, rank, dim_in]")
            adapters, rank = int(a.shape[0]), int(a.shape[1])
            _check("a", a, (adapters, rank, dim_in), dtype)
            _check("b", b, (adapters, dim_out, rank), dtype)
            if scale is not None:
                _check("scale", scale, (adapters,), _lib.F32)
        for name, t in (("w", w), ("a", a), ("b", b), ("scale", scale)):
            if t is None:
                continue
            if t.device.type != "cuda":
                raise VdbError(_lib.EINVAL, "%s is not on a GPU" % name)
            if t.device != w.device:
                raise VdbError(_lib.EINVAL, "%s is on %s, w on %s" % (name, t.device, w.device))
        self.w, self.a, self.b, self.scale = w, a, b, scale
        self.device = int(w.device.index or 0)
        self.dtype = dtype
        self.out_dtype = dtype if out_dtype is None else _dtype(out_dtype)
        if self.out_dtype not in (dtype, _lib.F32):
            raise VdbError(_lib.EINVAL, "out_dtype must be the weights' type or float32")
        self.dim_in, self.dim_out, self.groups, self.adapters, self.rank = dim_in, dim_out, groups, adapters, rank
        self.struct = _lib.ProjectionStruct(
            dim_in, dim_out, dtype, self.out_dtype, groups, adapters, rank, 0, w.data_ptr(),
            a.data_ptr() if a is not None else None, b.data_ptr() if b is not None else None,
            scale.data_ptr() if scale is not None else None)
        self.ptr = C.addressof(self.struct)
