"""Refusals of low-rank adapters that need no device."""
import ctypes

import numpy as np
import pytest

import welvet_amd as wv
from welvet_amd.adapters import AdapterBatch, AdapterRows, Adapters

OK = dict(rows=64, cols=64, max_rank=8, n_adapters=2, type="f16")


@pytest.mark.parametrize("bad,code,text", [
    (dict(rows=0), -2, "non-positive"), (dict(cols=-1), -2, "non-positive"), (dict(n_adapters=0), -2, "non-positive"),
    (dict(rows=(1 << 24) + 1), -2, "2^24"), (dict(cols=(1 << 24) + 1), -2, "2^24"),
    (dict(n_adapters=(1 << 20) + 1), -2, "2^20"), (dict(max_rank=0), -2, "max_rank 0"),
    (dict(max_rank=257), -2, "max_rank 257"), (dict(type=2), -3, "type 2"), (dict(type=-1), -3, "type -1"),
])
def test_create_refusals(bad, code, text):
    with pytest.raises(wv.WelvetError) as e:
        Adapters(**(OK | bad))
    assert e.value.code == code and text in str(e.value)


def test_nil_and_unknown():
    L = wv.lib()
    b, r, nb = AdapterBatch(1, 1, 0, 0), (AdapterRows * 5)(), ctypes.c_size_t()
    for i in range(5):
        r[i].adapters = 987654
    assert L.wv_adapters_create(None, None) == -1
    assert L.wv_adapters_free(987654) == -7
    assert L.wv_adapters_set(987654, 0, 0, 1.0, None, None) == -7
    assert L.wv_adapters_dev(ctypes.byref(b), None, 0, r, 1, None, 0, None) == -7
    assert b"unknown adapters" in L.wv_last_error()
    assert L.wv_adapters_dev(None, None, 0, r, 1, None, 0, None) == -1
    assert L.wv_adapters_dev(ctypes.byref(b), None, 0, r, 0, None, 0, None) == -2
    assert L.wv_adapters_dev(ctypes.byref(b), None, 0, r, 5, None, 0, None) == -2
    assert L.wv_adapters_scratch(ctypes.byref(b), r, 1, ctypes.byref(nb)) == -7


def test_python_checks():
    s = Adapters.__new__(Adapters)
    s.cfg = type("C", (), dict(rows=4, cols=6, type=0))
    for a, b in ((np.zeros((2, 5), np.float16), np.zeros((4, 2), np.float16)),
                 (np.zeros((2, 6), np.float16), np.zeros((3, 2), np.float16)),
                 (np.zeros((2, 6), np.float16), np.zeros((4, 3), np.float16)),
                 (np.zeros((2, 6), np.float32), np.zeros((4, 2), np.float16))):
        with pytest.raises(ValueError):
            s.set(0, a, b)
