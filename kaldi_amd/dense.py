"""Python mirror of the dense-layer operators over the C ABI (amlike_norm_*, amlike_linear_*,
amlike_convert_dev of include/amlike.h): root-mean-square norm with the residual's addition, matrix
product with bias, activation and residual, and conversion, in 32, 16 and 8 bits.  All arithmetic
happens in libamlike.so on the GPU; this file only marshals.

Types are "f32", "bf16", "f16" and "mx8" (e4m3 values with one e8m0 scale per 32 columns),
activations "none", "relu", "sigmoid", "tanh", "silu" and "gelu".
"""
import ctypes
from ctypes import POINTER, byref, c_float, c_void_p

import numpy as np

from . import _lib

TYPES = {"f32": 0, "bf16": 1, "f16": 2, "mx8": 3}
ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "silu": 4, "gelu": 5}


def _fp(a):
    return a.ctypes.data_as(POINTER(c_float)) if a is not None else None


def _int32(v, what):
    """v, where the C side takes 32 bits (ctypes would cut off the rest)."""
    if not -0x80000000 <= v < 0x80000000:
        raise ValueError("%s: %d does not fit 32 bits" % (what, v))
    return v


def _rows(a, cols, what):
    """A float32 [T x cols] array with contiguous rows, and its row stride in elements."""
    a = np.asarray(a, dtype=np.float32)
    if a.ndim != 2 or a.shape[1] != cols:
        raise ValueError("%s: shape %s, %d columns expected" % (what, a.shape, cols))
    _int32(a.shape[0], what)
    if a.strides[1] != 4 or a.strides[0] % 4 or not 4 * cols <= a.strides[0] < 4 * 0x80000000:
        a = np.ascontiguousarray(a)
    return a, a.strides[0] // 4 if a.shape[0] > 1 else cols


class Matrix:
    """Where a matrix lies in device memory: address, type, row stride in elements and, for "mx8",
    the scales' address and row stride in bytes (struct amlike_matrix).  Keeps no memory alive."""

    def __init__(self, ptr, type, ld, scales_ptr=0, ld_scales=0):
        if not (0 <= ptr < 1 << 64 and 0 <= scales_ptr < 1 << 64 and -1 << 63 <= ld < 1 << 63 and -1 << 63 <= ld_scales < 1 << 63):
            raise ValueError("Matrix: address or row stride out of range")
        self.c = _lib.Matrix(ptr, scales_ptr, ld, ld_scales, TYPES[type])
        self.ref = byref(self.c)


def _ref(m):
    return m.ref if m is not None else None


def ConvertDevice(x, rows, cols, out, stream=None):
    """out = x in out's type (amlike_convert_dev); x and out are Matrix."""
    if not (-0x80000000 <= rows < 0x80000000 and -0x80000000 <= cols < 0x80000000):
        _int32(rows, "rows"), _int32(cols, "cols")
    rc = _lib.lib().amlike_convert_dev(x.ref, rows, cols, out.ref, stream)
    if rc:
        _lib.check(rc)


class RmsNorm:
    """s = x + residual, out = s / sqrt(mean(s^2) + eps) * weight; weight [dim] or None (ones)."""

    def __init__(self, dim, weight=None, eps=1e-5, device=None):
        L = _lib.lib()
        _int32(int(dim), "dim")
        if device is not None:
            _lib.check(L.amlike_init(int(device)))
        w = None if weight is None else np.ascontiguousarray(weight, np.float32)
        if w is not None and w.shape != (dim,):
            raise ValueError("weight of %s for dim %d" % (w.shape, dim))
        self._h = c_void_p()
        _lib.check(L.amlike_norm_create(_fp(w), int(dim), float(eps), byref(self._h)))
        self._apply = L.amlike_norm_apply_dev

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().amlike_norm_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def Dim(self):
        return _lib.lib().amlike_norm_dim(self._h)

    def Apply(self, x, residual=None, return_sum=False):
        """Host arrays, fp32: the normalised rows, or (rows, sum)."""
        dim = self.Dim()
        x, ld = _rows(x, dim, "x")
        r, ldr = (None, 0) if residual is None else _rows(residual, dim, "residual")
        if r is not None and r.shape != x.shape:
            raise ValueError("residual of %s for x of %s" % (r.shape, x.shape))
        out = np.empty((x.shape[0], dim), np.float32)
        s = np.empty_like(out) if return_sum else None
        _lib.check(_lib.lib().amlike_norm_apply(self._h, _fp(x), ld, _fp(r), ldr, x.shape[0], _fp(s), dim, _fp(out), dim))
        return (out, s) if return_sum else out

    def ApplyDevice(self, x, rows, out, residual=None, sum=None, stream=None):
        """Matrix arguments, asynchronous on `stream` (amlike_norm_apply_dev)."""
        if not -0x80000000 <= rows < 0x80000000:
            _int32(rows, "rows")
        rc = self._apply(self._h, x.ref, _ref(residual), rows, _ref(sum), out.ref, stream)
        if rc:
            _lib.check(rc)


def linear_kernel_info(type, out, rows, input_dim, output_dim, aligned=True, units=256):
    """The kernel and form that Linear.ApplyDevice takes (amlike_linear_kernel_info); needs no GPU."""
    args = [_int32(v, "size") for v in (rows, input_dim, output_dim)]
    return _lib.lib().amlike_linear_kernel_info(TYPES[type], TYPES[out], *args, int(aligned), _int32(units, "units")).decode()


class Linear:
    """out = act(x weights^T + bias) + residual; weights [output x input], in `type` ("bf16", "f16", "mx8")."""

    def __init__(self, weights, bias=None, type="bf16", device=None):
        L = _lib.lib()
        if device is not None:
            _lib.check(L.amlike_init(int(device)))
        w = np.asarray(weights, np.float32)
        if w.ndim != 2:
            raise ValueError("weights of %s" % (w.shape,))
        w, ld = _rows(w, _int32(w.shape[1], "weights"), "weights")
        b = None if bias is None else np.ascontiguousarray(bias, np.float32)
        if b is not None and b.shape != (w.shape[0],):
            raise ValueError("bias of %s for %d outputs" % (b.shape, w.shape[0]))
        self._h = c_void_p()
        _lib.check(L.amlike_linear_create(_fp(w), ld, _fp(b), w.shape[1], w.shape[0], TYPES[type], byref(self._h)))
        self._apply = L.amlike_linear_apply_dev

    def close(self):
        if getattr(self, "_h", None):
            _lib.lib().amlike_linear_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def InputDim(self):
        return _lib.lib().amlike_linear_input_dim(self._h)

    def OutputDim(self):
        return _lib.lib().amlike_linear_output_dim(self._h)

    def Apply(self, x, activation="none", residual=None):
        """Host arrays, fp32; x is converted to the layer's type on the device."""
        x, ld = _rows(x, self.InputDim(), "x")
        n = self.OutputDim()
        r, ldr = (None, 0) if residual is None else _rows(residual, n, "residual")
        if r is not None and r.shape[0] != x.shape[0]:
            raise ValueError("residual of %s for %d rows" % (r.shape, x.shape[0]))
        out = np.empty((x.shape[0], n), np.float32)
        _lib.check(_lib.lib().amlike_linear_apply(self._h, _fp(x), ld, x.shape[0], ACTIVATIONS[activation], _fp(r), ldr,
                                                  _fp(out), n))
        return out

    def ApplyDevice(self, x, rows, out, activation="none", residual=None, stream=None):
        """Matrix arguments, asynchronous on `stream` (amlike_linear_apply_dev)."""
        if not -0x80000000 <= rows < 0x80000000:
            _int32(rows, "rows")
        rc = self._apply(self._h, x.ref, rows, ACTIVATIONS[activation], _ref(residual), out.ref, stream)
        if rc:
            _lib.check(rc)
