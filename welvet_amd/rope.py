"""Rotary positions (wv_rope_*): query and key rows turned to their positions, both
pair layouts, part of a head, scaled for contexts longer than the trained one."""
from __future__ import annotations

import ctypes

from . import check, lib

LAYOUTS = {"half": 0, "pairs": 1}  # WV_ROPE_HALF, WV_ROPE_PAIRS
SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp_dims": 3, "ramp_turns": 4}


class RopeConfig(ctypes.Structure):
    _fields_ = [("head_dim", ctypes.c_int32), ("rot_dim", ctypes.c_int32), ("layout", ctypes.c_int32),
                ("scaling", ctypes.c_int32), ("trained", ctypes.c_int32), ("theta", ctypes.c_double),
                ("factor", ctypes.c_double), ("low", ctypes.c_double),
                ("high", ctypes.c_double), ("gain", ctypes.c_double)]


class RopeRows(ctypes.Structure):
    _fields_ = [("d_x", ctypes.c_void_p), ("d_y", ctypes.c_void_p), ("x_stride", ctypes.c_int64),
                ("y_stride", ctypes.c_int64), ("n_heads", ctypes.c_int32)]


class Rope:
    """Owns a wv_rope handle; freed with free() or on GC. rot_dim None: the whole head."""

    handle = 0

    def __init__(self, head_dim: int, rot_dim: int | None = None, theta: float = 5e5, layout="half", scaling="none",
                 factor: float = 1.0, trained: int = 0, low: float = 1.0, high: float = 32.0, gain: float = 1.0):
        of = lambda x, names: names[x] if isinstance(x, str) else int(x)  # noqa: E731
        self.cfg = RopeConfig(head_dim, head_dim if rot_dim is None else rot_dim, of(layout, LAYOUTS),
                              of(scaling, SCALINGS), trained, theta, factor, low, high, gain)
        h = ctypes.c_uint64()
        check(lib().wv_rope_create(ctypes.byref(self.cfg), ctypes.byref(h)))
        self.handle = h.value

    def apply_dev(self, pos_ptr: int, n: int, q_ptr: int | None = None, n_heads: int = 0, k_ptr: int | None = None,
                  n_kv_heads: int = 0, *, q_stride: int = 0, k_stride: int = 0, q_out_ptr: int | None = None,
                  k_out_ptr: int | None = None, q_out_stride: int = 0, k_out_stride: int = 0,
                  stream: int | None = None) -> None:
        """n rows of q and of k (f32) turned to the positions pos (int32), in place unless an output is given."""
        q = RopeRows(q_ptr, q_out_ptr, q_stride, q_out_stride, n_heads)
        k = RopeRows(k_ptr, k_out_ptr, k_stride, k_out_stride, n_kv_heads)
        check(lib().wv_rope_dev(self.handle, pos_ptr, n, ctypes.byref(q), ctypes.byref(k), stream))

    def free(self) -> None:
        if self.handle:
            check(lib().wv_rope_free(self.handle))
            self.handle = 0

    def __del__(self):
        try:
            if self.handle:
                lib().wv_rope_free(self.handle)
                self.handle = 0
        except Exception:
            pass
