"""Lists of device arrays treated as one vector per instance: global norm, clipping, bounded steps (csrc/group.hip).

The counterpart for whole sets of messages of what damping does edge by edge: ``ExpectationPropagation.iterate(max_step=...)``
bounds the step of a sweep, new minus old over every message of the graph, with the operators of this module.
"""
import ctypes as C

import numpy as np

from .device import DeviceArray, dtype_code


class ArrayGroup:
    """Device arrays [batch, n_i] (or [n_i]) of one type and context, seen as ``batch`` instances: row b of every array.

    The arrays are kept as they are and must not overlap; lengths are free, also odd and zero.  Squares are summed in double:
    float64 components beyond 1e154 make a norm infinite, those below 1e-162 add nothing to it."""

    def __init__(self, arrays, ctx=None):
        arrays = list(arrays)
        if not arrays or not all(isinstance(a, DeviceArray) for a in arrays):
            raise ValueError("expected a list of one or more device arrays")
        self.ctx = ctx if ctx is not None else arrays[0].ctx
        self.dtype = arrays[0].dtype
        code = dtype_code(self.dtype)
        shapes = [a.shape if a.ndim == 2 else (1, a.size) for a in arrays if a.ndim in (1, 2)]
        if len(shapes) != len(arrays):
            raise ValueError("expected arrays [n] or [batch, n]")
        self.batch = shapes[0][0]
        for a, s in zip(arrays, shapes):
            if a.ctx is not self.ctx:
                raise ValueError("device array of another context")
            if a.dtype != self.dtype or s[0] != self.batch:
                raise ValueError(f"arrays of one list share type and batch: {self.dtype} x {self.batch} and {a.dtype} x {s[0]}")
        self.arrays, self.lengths = arrays, tuple(s[1] for s in shapes)
        k = len(arrays)
        h = C.c_void_p()
        self._handle = None
        self.ctx._call("tramp_group_create", code, k, (C.c_void_p * k)(*[a.ptr for a in arrays]),
                       (C.c_size_t * k)(*self.lengths), self.batch, C.byref(h))
        self._handle = h

    def __del__(self):
        try:
            self.ctx.release("tramp_group_destroy", self._handle)
        except Exception:
            pass
        self._handle = None

    def __len__(self):
        return len(self.arrays)

    def _norm(self, norm):
        if norm is None:
            return self.ctx.empty((self.batch,), np.float64)
        if not isinstance(norm, DeviceArray) or norm.ctx is not self.ctx or norm.dtype != np.float64 or norm.size != self.batch:
            raise ValueError(f"norm needs a device array of {self.batch} float64 in this context, got {norm!r}")
        return norm

    def _list(self, other, what):
        if not isinstance(other, ArrayGroup) or other.ctx is not self.ctx:
            raise ValueError(f"{what} must be an ArrayGroup of the same context")
        if other.dtype != self.dtype or other.batch != self.batch or other.lengths != self.lengths:
            raise ValueError(f"{what} must hold arrays of the same type, batch and lengths")
        return other

    @staticmethod
    def _bound(value, what):
        value = float(value)
        if not value > 0.0:
            raise ValueError(f"{what} must be positive, got {value}")
        return value

    def norm(self, out=None):
        "double[batch]: the root of the sum of squares over all arrays"
        out = self._norm(out)
        self.ctx._call("tramp_group_norm", self._handle, out.ptr)
        return out

    def clip(self, max_norm, out=None, norm=None):
        """Every array times min(1, max_norm / norm) per instance, in place or into the arrays of ``out``; returns the norms
        before.  An instance whose norm is infinite or NaN stays as it is."""
        dst = self if out is None else self._list(out, "out")
        norm = self._norm(norm)
        self.ctx._call("tramp_group_clip", self._handle, self._bound(max_norm, "max_norm"), dst._handle, norm.ptr)
        return norm

    def limit_step(self, prev, max_step, out=None, norm=None, a=None, a_prev=None, refresh=False):
        """prev + min(1, max_step / |x - prev|) (x - prev) per instance, in place or into ``out``; returns the norms |x - prev|.
        ``a``, ``a_prev`` (double[..., batch]): precisions moved by the same factor, in place in ``a``.  ``refresh``: the result
        is written over ``prev`` (and ``a_prev``) as well.  A step that is infinite or NaN is taken whole."""
        prev = self._list(prev, "prev")
        dst = self if out is None else self._list(out, "out")
        norm = self._norm(norm)
        n_a = 0
        if (a is None) != (a_prev is None):
            raise ValueError("a and a_prev come together")
        if a is not None:
            for t in (a, a_prev):
                if not isinstance(t, DeviceArray) or t.ctx is not self.ctx or t.dtype != np.float64 or t.shape[-1] != self.batch or t.size != a.size:
                    raise ValueError(f"a and a_prev must be float64 device arrays [..., {self.batch}] of one size")
            n_a = a.size // self.batch
        self.ctx._call("tramp_group_limit_step", self._handle, prev._handle, self._bound(max_step, "max_step"), dst._handle,
                       int(bool(refresh)), n_a, a.ptr if n_a else None, a_prev.ptr if n_a else None, norm.ptr)
        return norm


__all__ = ["ArrayGroup"]
