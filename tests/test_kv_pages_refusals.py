"""Refusals of the calls on a page table that need no device."""
import ctypes

import welvet_amd as wv
from welvet_amd.kv import KVBatch, KVTables


def test_unknown_cache():
    L = wv.lib()
    t, b, nb = KVTables(1, 1, 0, 0, 0, 0), KVBatch(1, 1, 1, 0, 0, 0), ctypes.c_size_t()
    assert L.wv_kv_tables_work(987654, 1, 1, ctypes.byref(nb)) == -7
    assert L.wv_kv_fork_dev(987654, ctypes.byref(t), None, None) == -7
    assert L.wv_kv_resize_dev(987654, ctypes.byref(t), None, None, None) == -7
    assert L.wv_kv_compact_dev(987654, ctypes.byref(t), None, None) == -7
    assert L.wv_kv_copy_pages_dev(987654, None, None, 0, None) == -7
    assert L.wv_kv_slots_dev(987654, ctypes.byref(b), None, None, None) == -7
    assert b"unknown cache" in L.wv_last_error()
