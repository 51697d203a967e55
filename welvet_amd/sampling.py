"""Draws next tokens from logits on the device (wv_sample_dev): temperature, top-k,
top-p and min-p per row, from the caller's uniform numbers."""
from __future__ import annotations

import ctypes

from . import check, lib


class Sampling(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_void_p), ("top_k", ctypes.c_void_p), ("top_p", ctypes.c_void_p),
                ("min_p", ctypes.c_void_p), ("uniform", ctypes.c_void_p)]


def sample_dev(logits_ptr: int, rows: int, vocab: int, tokens_ptr: int, uniform_ptr: int, *, stride: int = 0,
               temperature_ptr: int | None = None, top_k_ptr: int | None = None, top_p_ptr: int | None = None,
               min_p_ptr: int | None = None, probs_ptr: int | None = None, stream: int | None = None) -> None:
    """tokens[r] (int32) of each row of f32 logits; the settings are device arrays of one value per row
    (float, top_k int32), None leaves a step out. probs (float): the drawn token's share of what was kept."""
    s = Sampling(temperature_ptr, top_k_ptr, top_p_ptr, min_p_ptr, uniform_ptr)
    check(lib().wv_sample_dev(logits_ptr, stride, rows, vocab, ctypes.byref(s), tokens_ptr, probs_ptr, stream))
