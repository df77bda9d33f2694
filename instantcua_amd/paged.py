"""Paged K/V caches: several sequences in one pool of pages (the ``icua_paged_*`` calls of
``include/icua.h``).

``PagedCache`` is one layer's pool.  ``store`` normalises, rotates and writes new tokens, ``attention``
runs every sequence's new tokens over its slots, ``load`` reads slots back.  Buffers are anything with
a device address ``ptr`` (``engine.DeviceBuffer``).  The calls enqueue on ``stream`` (a hipStream_t as
an integer, 0: the null stream) and return without waiting; ``engine.lib().icua_device_sync`` or a copy
to the host waits.  Errors raise ``EngineError``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from .engine import HD, DeviceBuffer, EngineError, _check, lib
from .modelfile import WeightFormat, matrix_bytes

F32, F16 = 0, 1


class _Pages(C.Structure):
    _fields_ = [("fmt", C.c_int32), ("n_kv", C.c_int32), ("page_slots", C.c_int32), ("n_pages", C.c_int32),
                ("k", C.c_void_p), ("v", C.c_void_p), ("k_scales", C.c_void_p), ("v_scales", C.c_void_p)]


class _Store(C.Structure):
    _fields_ = [("type", C.c_int32), ("q_type", C.c_int32), ("n_tokens", C.c_int32), ("n_heads", C.c_int32),
                ("qkv", C.c_void_p), ("qkv_stride", C.c_int64), ("q", C.c_void_p), ("q_stride", C.c_int64),
                ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("eps", C.c_float), ("rope", C.c_void_p),
                ("rope_rows", C.c_int32), ("rot_dim", C.c_int32), ("interleaved", C.c_int32), ("pos", C.c_void_p),
                ("slots", C.c_void_p)]


class _Attention(C.Structure):
    _fields_ = [("type", C.c_int32), ("n_heads", C.c_int32), ("n_seqs", C.c_int32), ("n_tokens", C.c_int32),
                ("max_q", C.c_int32), ("max_kv", C.c_int32), ("scale", C.c_float), ("q", C.c_void_p),
                ("q_stride", C.c_int64), ("out", C.c_void_p), ("out_stride", C.c_int64), ("q_start", C.c_void_p),
                ("kv_len", C.c_void_p), ("tables", C.c_void_p), ("table_width", C.c_int32), ("work", C.c_void_p),
                ("work_bytes", C.c_size_t)]


class _Load(C.Structure):
    _fields_ = [("type", C.c_int32), ("n_rows", C.c_int32), ("slots", C.c_void_p), ("k", C.c_void_p),
                ("v", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


def _ptr(b):
    return None if b is None else b.ptr


class PagedCache:
    """A pool of ``n_pages`` pages of ``page_slots`` slots for ``n_kv`` KV heads, fp16 or q8.  Its
    buffers are allocated (their contents undefined) unless given."""

    def __init__(self, fmt: int, n_kv: int, page_slots: int, n_pages: int, k=None, v=None, k_scales=None,
                 v_scales=None):
        if fmt not in (WeightFormat.F16, WeightFormat.Q8):
            raise EngineError("a paged cache is f16 or q8")
        if min(n_kv, page_slots, n_pages) < 1:
            raise EngineError("a paged cache has at least one KV head, slot and page")
        self.fmt, self.n_kv, self.page_slots, self.n_pages = int(fmt), n_kv, page_slots, n_pages
        need = matrix_bytes(fmt, n_pages * n_kv * page_slots, HD)
        buffers = []
        for b, n in ((k, need[0]), (v, need[0]), (k_scales, need[1]), (v_scales, need[1])):
            if n and b is None:
                b = DeviceBuffer(n)
            if n and b.nbytes < n:
                raise EngineError(f"a buffer of the pool has {b.nbytes} bytes, not {n}")
            buffers.append(b if n else None)
        self.k, self.v, self.k_scales, self.v_scales = buffers
        self._pages = _Pages(self.fmt, n_kv, page_slots, n_pages, *(_ptr(b) for b in buffers))
        self._at = C.addressof(self._pages)

    def slots(self, table: Sequence[int], first: int, count: int) -> np.ndarray:
        """Pool slots of slots first .. first + count - 1 of a sequence with these pages."""
        p = np.arange(first, first + count)
        pages = np.asarray(table, dtype=np.int64)
        if first < 0 or count < 0 or first + count > pages.size * self.page_slots:
            raise EngineError("the slots lie outside the table's pages")
        out = pages[p // self.page_slots] * self.page_slots + p % self.page_slots
        if count and (out.min() < 0 or out.max() >= self.n_pages * self.page_slots):
            raise EngineError("a page of the table lies outside the pool")
        return out.astype(np.int32)

    def store(self, qkv, n_tokens: int, slots, n_heads: int = 0, q=None, q_norm=None, k_norm=None, rope=None,
              rope_rows: int = 0, pos=None, rot_dim: Optional[int] = None, interleaved: bool = False,
              eps: float = 1e-6, type: int = F32, q_type: int = F32, qkv_stride: int = 0, q_stride: int = 0,
              stream: int = 0) -> None:
        """icua_paged_store; without a table (``rope``) nothing is rotated, with one all of a head
        unless ``rot_dim`` says less."""
        if rot_dim is None:
            rot_dim = 0 if rope is None else HD
        a = _Store(type, q_type, n_tokens, n_heads, _ptr(qkv), qkv_stride, _ptr(q), q_stride, _ptr(q_norm),
                   _ptr(k_norm), eps, _ptr(rope), rope_rows, rot_dim, interleaved, _ptr(pos), _ptr(slots))
        _check(lib().icua_paged_store(self._at, C.addressof(a), stream))

    def attention_work(self, n_heads: int, n_seqs: int, n_tokens: int, table_width: Optional[int] = None,
                       max_q: int = 0, max_kv: int = 0) -> int:
        """Bytes of workspace for an attention call of exactly these sizes; without ``table_width`` the table is
        taken to be as wide as ``max_kv`` slots need, or one page if that is 0 too (a call without a bound on
        slots over wider tables has to say their width here)."""
        if table_width is None:
            table_width = max(1, -(-max_kv // self.page_slots))
        a = _Attention(0, n_heads, n_seqs, n_tokens, max_q, max_kv, 0.0, table_width=table_width)
        n = C.c_size_t()
        _check(lib().icua_paged_attention_work(self._at, C.addressof(a), C.byref(n)))
        return n.value

    def attention(self, q, out, n_heads: int, q_start, kv_len, tables, n_seqs: int, n_tokens: int, table_width: int,
                  max_q: int = 0, max_kv: int = 0, scale: float = 0.0, type: int = F32, q_stride: int = 0,
                  out_stride: int = 0, work=None, stream: int = 0) -> None:
        """icua_paged_attention; ``work`` has ``attention_work`` bytes (None where that is 0)."""
        a = _Attention(type, n_heads, n_seqs, n_tokens, max_q, max_kv, scale, _ptr(q), q_stride, _ptr(out),
                       out_stride, _ptr(q_start), _ptr(kv_len), _ptr(tables), table_width, _ptr(work),
                       0 if work is None else work.nbytes)
        _check(lib().icua_paged_attention(self._at, C.addressof(a), stream))

    def load(self, slots, n_rows: int, k=None, v=None, type: int = F32, token_stride: int = 0, head_stride: int = 0,
             stream: int = 0) -> None:
        """icua_paged_load."""
        a = _Load(type, n_rows, _ptr(slots), _ptr(k), _ptr(v), token_stride, head_stride)
        _check(lib().icua_paged_load(self._at, C.addressof(a), stream))
