"""Refusals of wv_sample_dev that need no device."""
import ctypes

import welvet_amd as wv
from welvet_amd.sampling import Sampling


def test_refusals_without_device():
    L = wv.lib()
    s = Sampling(None, None, None, None, 16)
    none = Sampling(None, None, None, None, None)
    by = ctypes.byref(s)
    assert L.wv_sample_dev(16, 0, 1, 100, None, 16, None, None) == -1
    assert L.wv_sample_dev(16, 0, -1, 100, by, 16, None, None) == -2
    assert L.wv_sample_dev(16, 0, 1, 0, by, 16, None, None) == -2
    assert L.wv_sample_dev(16, 0, 1, (1 << 19) + 1, by, 16, None, None) == -2
    assert L.wv_sample_dev(16, 0, (1 << 20) + 1, 100, by, 16, None, None) == -2
    assert L.wv_sample_dev(16, 99, 1, 100, by, 16, None, None) == -2
    assert b"stride" in L.wv_last_error()
    assert L.wv_sample_dev(None, 0, 1, 100, by, 16, None, None) == -1
    assert L.wv_sample_dev(16, 0, 1, 100, by, None, None, None) == -1
    assert L.wv_sample_dev(16, 0, 1, 100, ctypes.byref(none), 16, None, None) == -1
    assert L.wv_sample_dev(None, 0, 0, 100, by, None, None, None) == 0
