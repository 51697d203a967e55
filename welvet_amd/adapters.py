"""Low-rank adapters of many requests beside a shared projection (wv_adapters_*):
y = base + scale B (A x) with each sequence's own A, B and scale, for up to four
projections of the same rows in one call."""
from __future__ import annotations

import ctypes

import numpy as np

from . import check, lib

TYPES = {"f16": 0, "bf16": 1}  # WV_ADAPTER_*


class AdaptersConfig(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int32), ("cols", ctypes.c_int32), ("max_rank", ctypes.c_int32),
                ("n_adapters", ctypes.c_int32), ("type", ctypes.c_int32)]


class AdapterBatch(ctypes.Structure):
    """wv_adapter_batch: sequence b owns token rows cu_q[b] .. cu_q[b+1]-1 of n_tokens and adapter[b] (-1: none).
    max_q (most tokens of one sequence, 0: unknown) only steers the launch. The arrays are int32 on the device and
    have to live until the work is done."""
    _fields_ = [("n_seqs", ctypes.c_int32), ("n_tokens", ctypes.c_int32), ("max_q", ctypes.c_int32),
                ("d_cu_q", ctypes.c_void_p), ("d_adapter", ctypes.c_void_p)]

    def __init__(self, n_seqs: int, n_tokens: int, cu_q_ptr: int, adapter_ptr: int, max_q: int = 0):
        super().__init__(n_seqs, n_tokens, max_q, cu_q_ptr, adapter_ptr)


class AdapterRows(ctypes.Structure):
    _fields_ = [("adapters", ctypes.c_uint64), ("d_y", ctypes.c_void_p), ("d_base", ctypes.c_void_p),
                ("y_stride", ctypes.c_int64), ("base_stride", ctypes.c_int64)]


class Adapters:
    """Owns a wv_adapters handle, the adapters of one projection; freed with free() or on GC."""

    handle = 0

    def __init__(self, rows: int, cols: int, max_rank: int, n_adapters: int, type="bf16"):
        t = TYPES[type] if isinstance(type, str) else int(type)
        self.cfg = AdaptersConfig(rows, cols, max_rank, n_adapters, t)
        h = ctypes.c_uint64()
        check(lib().wv_adapters_create(ctypes.byref(self.cfg), ctypes.byref(h)))
        self.handle = h.value

    def set(self, index: int, a: np.ndarray, b: np.ndarray, scale: float = 1.0) -> None:
        """Adapter `index`: a [rank, cols] and b [rows, rank], as float16 or as the bits (uint16) of the set's type."""
        bits = []
        for x, want in ((a, (None, self.cfg.cols)), (b, (self.cfg.rows, None))):
            x = np.ascontiguousarray(x)
            if x.dtype == np.float16 and self.cfg.type == 0:
                x = x.view(np.uint16)
            if x.dtype != np.uint16 or x.ndim != 2 or any(w not in (None, n) for n, w in zip(x.shape, want)):
                raise ValueError(f"Adapters.set: {x.dtype} {x.shape}, want 16-bit floats of {want}")
            bits.append(x)
        if bits[0].shape[0] != bits[1].shape[1]:
            raise ValueError(f"Adapters.set: ranks {bits[0].shape[0]} and {bits[1].shape[1]}")
        check(lib().wv_adapters_set(self.handle, index, bits[0].shape[0], scale, bits[0].ctypes.data,
                                    bits[1].ctypes.data))

    def unset(self, index: int) -> None:
        check(lib().wv_adapters_set(self.handle, index, 0, 1.0, None, None))

    def free(self) -> None:
        if self.handle:
            check(lib().wv_adapters_free(self.handle))
            self.handle = 0

    def __del__(self):
        try:
            if self.handle:
                lib().wv_adapters_free(self.handle)
                self.handle = 0
        except Exception:
            pass


def _rows(sets, y_ptrs, base_ptrs, y_strides, base_strides):
    n = len(sets)
    for x in (y_ptrs, base_ptrs, y_strides, base_strides):
        if x is not None and len(x) != n:
            raise ValueError(f"adapters: {n} sets, {len(x)} pointers or strides")
    rows = (AdapterRows * n)()
    for i in range(n):
        r = rows[i]
        r.adapters = sets[i].handle
        if y_ptrs is not None:
            r.d_y = y_ptrs[i]
        if base_ptrs is not None:
            r.d_base = base_ptrs[i]
        if y_strides is not None:
            r.y_stride = y_strides[i]
        if base_strides is not None:
            r.base_stride = base_strides[i]
    return rows


def apply_dev(sets, batch: AdapterBatch, x_ptr: int, y_ptrs, *, base_ptrs=None, x_stride: int = 0, y_strides=None,
              base_strides=None, scratch_ptr: int | None = None, scratch_bytes: int = 0,
              stream: int | None = None) -> None:
    """y = base + scale B (A x) for each set (base None: y itself), rows of f32; one pointer and stride a set."""
    rows = _rows(sets, y_ptrs, base_ptrs, y_strides, base_strides)
    check(lib().wv_adapters_dev(ctypes.byref(batch), x_ptr, x_stride, rows, len(sets), scratch_ptr, scratch_bytes,
                                stream))


def scratch(sets, batch: AdapterBatch) -> int:
    """Bytes of scratch a call may be given (and has to be under graph capture)."""
    nb = ctypes.c_size_t()
    check(lib().wv_adapters_scratch(ctypes.byref(batch), _rows(sets, None, None, None, None), len(sets),
                                    ctypes.byref(nb)))
    return nb.value
