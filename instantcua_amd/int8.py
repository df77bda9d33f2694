"""Products on 8-bit integers with a scale for each token and each output channel (the ``icua_i8_*`` calls of
``include/icua.h``).

``quantize`` makes the codes and scales of rows: of a batch's tokens, normalised on the way, or of a matrix's output
channels.  ``matmul`` multiplies tokens by a matrix, with a residual added or as silu(gate) * up of two.  Buffers are
anything with a device address ``ptr`` (``engine.DeviceBuffer``).  The calls enqueue on ``stream`` (a hipStream_t as
an integer, 0: the null stream) and return without waiting; ``engine.lib().icua_device_sync`` or a copy to the host
waits.  Errors raise ``EngineError``.
"""
from __future__ import annotations

import ctypes as C

from .engine import _check, lib

F32, F16 = 0, 1


class _Quantize(C.Structure):
    _fields_ = [("type", C.c_int32), ("n_rows", C.c_int32), ("n_cols", C.c_int32), ("x", C.c_void_p),
                ("x_stride", C.c_int64), ("norm", C.c_void_p), ("eps", C.c_float), ("codes", C.c_void_p),
                ("codes_stride", C.c_int64), ("scales", C.c_void_p)]


class _Matmul(C.Structure):
    _fields_ = [("type", C.c_int32), ("gated", C.c_int32), ("n_rows", C.c_int32), ("n_out", C.c_int32),
                ("n_in", C.c_int32), ("x", C.c_void_p), ("x_stride", C.c_int64), ("x_scales", C.c_void_p),
                ("w", C.c_void_p), ("w_stride", C.c_int64), ("w_scales", C.c_void_p), ("add", C.c_void_p),
                ("add_stride", C.c_int64), ("y", C.c_void_p), ("y_stride", C.c_int64), ("work", C.c_void_p),
                ("work_bytes", C.c_size_t)]


def _ptr(b):
    return None if b is None else b.ptr


def quantize(x, codes, scales, n_rows: int, n_cols: int, norm=None, eps: float = 1e-6, type: int = F32,
             x_stride: int = 0, codes_stride: int = 0, stream: int = 0) -> None:
    """icua_i8_quantize."""
    a = _Quantize(type, n_rows, n_cols, _ptr(x), x_stride, _ptr(norm), eps, _ptr(codes), codes_stride, _ptr(scales))
    _check(lib().icua_i8_quantize(C.addressof(a), stream))


def matmul_work(n_rows: int, n_out: int, n_in: int, gated: bool = False) -> int:
    """Bytes of workspace for a product of exactly these sizes."""
    a = _Matmul(F32, gated, n_rows, n_out, n_in)
    n = C.c_size_t()
    _check(lib().icua_i8_matmul_work(C.addressof(a), C.byref(n)))
    return n.value


def matmul(x, x_scales, w, w_scales, y, n_rows: int, n_out: int, n_in: int, add=None, gated: bool = False,
           type: int = F32, x_stride: int = 0, w_stride: int = 0, add_stride: int = 0, y_stride: int = 0, work=None,
           stream: int = 0) -> None:
    """icua_i8_matmul; ``work`` has ``matmul_work`` bytes (None where that is 0)."""
    a = _Matmul(type, gated, n_rows, n_out, n_in, _ptr(x), x_stride, _ptr(x_scales), _ptr(w), w_stride, _ptr(w_scales),
                _ptr(add), add_stride, _ptr(y), y_stride, _ptr(work), 0 if work is None else work.nbytes)
    _check(lib().icua_i8_matmul(C.addressof(a), stream))
