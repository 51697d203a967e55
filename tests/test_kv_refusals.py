"""Refusals of the paged KV cache that need no device: sizes, types, handles."""
import ctypes

import pytest

import welvet_amd as wv
from welvet_amd.kv import KVBatch, KVCache

OK = dict(n_layers=1, n_kv_heads=2, head_dim=64, page_size=32, n_pages=4, type="q8")


@pytest.mark.parametrize("bad,code,text", [
    (dict(n_layers=0), -2, "non-positive"),
    (dict(n_kv_heads=-1), -2, "non-positive"),
    (dict(n_pages=0), -2, "non-positive"),
    (dict(head_dim=96), -2, "head_dim 96"),
    (dict(page_size=16), -2, "page_size 16"),
    (dict(page_size=48), -2, "page_size 48"),
    (dict(page_size=512), -2, "page_size 512"),
    (dict(type=2), -3, "type 2"),
    (dict(type=-1), -3, "type -1"),
    (dict(n_kv_heads=5000), -2, "KV heads"),
    (dict(n_pages=1 << 26), -2, "2^31"),
    (dict(n_layers=(1 << 31) - 1, n_kv_heads=4096, head_dim=128, n_pages=(1 << 26) - 1, type="f16"), -4, "layers"),
])
def test_create_refusals(bad, code, text):
    with pytest.raises(wv.WelvetError) as e:
        KVCache(**(OK | bad))
    assert e.value.code == code and text in str(e.value)


def test_create_nil():
    L = wv.lib()
    assert L.wv_kv_create(None, None) == -1


def test_unknown_handles():
    L = wv.lib()
    b = KVBatch(1, 1, 1, 0, 0, 0)
    nb = ctypes.c_size_t()
    assert L.wv_kv_free(987654) == -7
    assert L.wv_kv_info(987654, None, None) == -7
    assert L.wv_kv_write_dev(987654, 0, None, None, 0, 0, None, 0, None) == -7
    assert L.wv_kv_read_dev(987654, 0, None, 0, None, None, 0, 0, None) == -7
    assert L.wv_kv_attention_dev(987654, 0, ctypes.byref(b), None, 0, 2, 1.0, 0, None, 0, None, 0, None) == -7
    assert L.wv_kv_attention_scratch(987654, ctypes.byref(b), 2, 0, ctypes.byref(nb)) == -7
    assert b"unknown cache" in L.wv_last_error()
