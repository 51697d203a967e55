"""Paged KV cache (wv_kv_*): the K and V rows of many sequences in one pool of
pages, as fp16 or int8 codes with a scale per position and KV head, and the
attention of new tokens over it. Rows, tables and results are device pointers."""
from __future__ import annotations

import ctypes

from . import check, lib

TYPES = {"f16": 0, "q8": 1}  # WV_KV_*


class KVConfig(ctypes.Structure):
    _fields_ = [("n_layers", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("n_pages", ctypes.c_int32), ("type", ctypes.c_int32)]


class KVBatch(ctypes.Structure):
    """wv_kv_batch: sequence b owns query rows cu_q[b] .. cu_q[b+1]-1 of n_tokens and keys 0 .. kv_len[b]-1,
    key j in page pages[b][j // page_size]. max_q (most new tokens of one sequence, 0: unknown) only steers
    the launch. The arrays are int32 on the device and have to live until the work is done."""
    _fields_ = [("n_seqs", ctypes.c_int32), ("n_tokens", ctypes.c_int32), ("max_pages", ctypes.c_int32),
                ("max_q", ctypes.c_int32), ("d_cu_q", ctypes.c_void_p), ("d_kv_len", ctypes.c_void_p),
                ("d_pages", ctypes.c_void_p)]

    def __init__(self, n_seqs: int, n_tokens: int, max_pages: int, cu_q_ptr: int, kv_len_ptr: int, pages_ptr: int,
                 max_q: int = 0):
        super().__init__(n_seqs, n_tokens, max_pages, max_q, cu_q_ptr, kv_len_ptr, pages_ptr)


class KVCache:
    """Owns a wv_kv cache handle; freed with free() or on GC."""

    handle = 0

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, page_size: int, n_pages: int, type="q8"):
        t = TYPES[type] if isinstance(type, str) else int(type)
        self.cfg = KVConfig(n_layers, n_kv_heads, head_dim, page_size, n_pages, t)
        h = ctypes.c_uint64()
        check(lib().wv_kv_create(ctypes.byref(self.cfg), ctypes.byref(h)))
        self.handle = h.value

    def info(self):
        cfg, nb = KVConfig(), ctypes.c_size_t()
        check(lib().wv_kv_info(self.handle, ctypes.byref(cfg), ctypes.byref(nb)))
        return {name: getattr(cfg, name) for name, _ in KVConfig._fields_} | {"device_bytes": nb.value}

    def write_dev(self, layer: int, k_ptr: int, v_ptr: int, slots_ptr: int, n: int, k_stride: int = 0,
                  v_stride: int = 0, stream: int | None = None) -> None:
        """n rows of K and V (f32) into the positions slots_ptr (int64); slots outside the pool are skipped."""
        check(lib().wv_kv_write_dev(self.handle, layer, k_ptr, v_ptr, k_stride, v_stride, slots_ptr, n, stream))

    def read_dev(self, layer: int, slots_ptr: int, n: int, k_ptr: int, v_ptr: int, k_stride: int = 0,
                 v_stride: int = 0, stream: int | None = None) -> None:
        """n positions back as f32 rows; slots outside the pool read 0."""
        check(lib().wv_kv_read_dev(self.handle, layer, slots_ptr, n, k_ptr, v_ptr, k_stride, v_stride, stream))

    def attention_dev(self, layer: int, batch: KVBatch, q_ptr: int, out_ptr: int, n_heads: int, scale: float,
                      window: int = 0, q_stride: int = 0, out_stride: int = 0, scratch_ptr: int | None = None,
                      scratch_bytes: int = 0, stream: int | None = None) -> None:
        """Causal attention of the batch's new tokens (f32 rows of n_heads heads) over their cached keys."""
        check(lib().wv_kv_attention_dev(self.handle, layer, ctypes.byref(batch), q_ptr, q_stride, n_heads, scale,
                                        window, out_ptr, out_stride, scratch_ptr, scratch_bytes, stream))

    def attention_scratch(self, batch: KVBatch, n_heads: int, window: int = 0) -> int:
        """Bytes of scratch an attention call may be given (needed only for calls under graph capture)."""
        nb = ctypes.c_size_t()
        check(lib().wv_kv_attention_scratch(self.handle, ctypes.byref(batch), n_heads, window, ctypes.byref(nb)))
        return nb.value

    def free(self) -> None:
        if self.handle:
            check(lib().wv_kv_free(self.handle))
            self.handle = 0

    def __del__(self):
        try:
            if self.handle:
                lib().wv_kv_free(self.handle)
                self.handle = 0
        except Exception:
            pass
