"""Attention over the paged cache where values, keys or queries lie far from 1, and that a row's bits come from the
keys it attends alone: row and tile kernel, whole and cut into key ranges."""
import ctypes

import numpy as np
import pytest
import torch

import welvet_amd as wv
from kv_ref import stored
from test_gpu_kv import Pool, dev, rows
from welvet_amd.kv import KVBatch, KVCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


# heads, kv heads, hd, keys, new tokens, cut into key ranges
ROW = [(8, 2, 128, 1, 1, False), (8, 2, 128, 40, 1, False), (8, 2, 64, 300, 40, False), (4, 1, 128, 9001, 1, True)]
TILE = [(64, 16, 64, 1900, 1900, False), (32, 8, 128, 4200, 515, True)]


def reference(q, k, v, n, scale, window=0):
    """The rows in float64 over held K and V, and what each value may be off by: a score by
    d = (2^-21 + (hd + 2) 2^-24) scale sum|q k| (fp16 pairs, hd products summed in f32, two scales), an exponential by
    a relative d + 2^-21, sums over L keys and their quotient by L 2^-24 each; the fp16 pair of a probability times
    its V scale also by 2^-25 in units of 2^-14 of the largest scale that the ROW attends: 2^-37 of its largest |V|
    per key. 2^-149 for results that are subnormal."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    H, hd, L = q.shape[1], q.shape[2], k.shape[0]
    G = H // k.shape[1]
    pos, key = L - n + np.arange(n)[:, None], np.arange(L)[None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(H):
        kk, vv = k[:, h // G], v[:, h // G]
        s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h] = w @ vv
        big = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T * scale, 0.0).max(1, keepdims=True)
        d = (2.0 ** -21 + (hd + 2) * 2.0 ** -24) * big + 2.0 ** -21 + L * 2.0 ** -24
        top = np.where(seen, np.abs(vv).max(1)[None], 0.0).max(1, keepdims=True)
        tol[:, h] = 2 * d * (w @ np.abs(vv)) + L * 2.0 ** -37 * top + 2.0 ** -149
    return out, tol


def close(got, p, n, scale, window=0, only=slice(None)):
    ref, tol = reference(p.q, stored(p.k[0], p.typ), stored(p.v[0], p.typ), n, np.float64(np.float32(scale)), window)
    off = np.abs(got.astype(np.float64) - ref)[only]
    assert np.isfinite(got[only]).all(), f"{(~np.isfinite(got[only])).sum()} values not finite"
    bad = off > tol[only]
    assert not bad.any(), f"{bad.sum()} values, by up to {(off / tol[only]).max():.3g} of the bound"


def pool(seed, typ, shape):
    heads, kvh, hd, kv, new, cut = shape
    p = Pool(np.random.default_rng(seed), [kv], kvh, hd, 64, typ)
    assert (p.kv.attention_scratch(KVBatch(1, new, p.width, 0, 0, 0, max_q=new), heads) > 0) == cut
    return p


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("shape", ROW + TILE)
@pytest.mark.parametrize("even", [False, True])
def test_large_values(typ, shape, even):
    """V up to the end of the range: the sums of the weights' multiples of it never lie above the largest |V|."""
    heads, kvh, hd, kv, new, _ = shape
    p = pool(41, typ, shape)
    if even:  # equal weights, one sign: the mean of values next to f32's largest
        p.k[0][:] = 0
        p.v[0] = np.float32(3e38) * (1 - np.abs(p.v[0]) * np.float32(0.01))
    else:
        p.v[0] *= np.float32(2e37)
    p.fill()
    close(p.attend([new], heads, max_q=new), p, new, 1 / np.sqrt(hd))


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("shape", ROW + TILE)
def test_small_values(typ, shape):
    """V rows next to 2^-100, equal weights, one sign: a mean that loses nothing on the way. Every weight is exactly
    2^14 and its scale at most split in 22 bits; two sums for every 16 keys, roundings of 2^-24 each, and 8 more."""
    heads, kvh, hd, kv, new, _ = shape
    p = pool(42, typ, shape)
    p.k[0][:] = 0
    p.v[0] = np.float32(2.0 ** -99) * (1 + np.abs(p.v[0]) / 8)
    p.fill()
    got = p.attend([new], heads, max_q=new).astype(np.float64)
    v = np.repeat(stored(p.v[0], typ), heads // kvh, 1)
    ref = (np.cumsum(v, 0) / np.arange(1, kv + 1)[:, None, None])[kv - new:]
    off = np.abs(got - ref).max() / np.abs(ref).max()
    assert off <= 2.0 ** -22 + (kv / 8 + 8) * 2.0 ** -24, off


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("shape", ROW + TILE)
@pytest.mark.parametrize("key,query,factor", [(1e33, 1e-33, 1), (1e36, 1e-36, 1), (1e-29, 1e29, 1), (1e35, 1, 1e-35),
                                              (1e36, 1e-20, 1e-16), (1e-20, 1e-15, 1e35), (1e-29, 1e36, 1e-7)])
def test_scores_of_large_and_small_factors(typ, shape, key, query, factor):
    """Keys, queries and the scale far from 1, their product and so the scores ordinary."""
    heads, kvh, hd, kv, new, _ = shape
    p = pool(43, typ, shape)
    p.k[0] *= np.float32(key)
    p.fill()
    q = rows(p.rng, new, heads, hd) * np.float32(query)
    scale = factor / np.sqrt(hd)
    close(p.attend([new], heads, max_q=new, q=q, scale=scale), p, new, scale)


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("shape", [(8, 2, 128, 300, 12), (8, 2, 64, 300, 40), (32, 8, 128, 4200, 515),
                                   (64, 16, 64, 1900, 1900)])
@pytest.mark.parametrize("power", [3, 20, 110])
@pytest.mark.parametrize("left", [False, True])
def test_rows_come_from_their_own_keys(typ, shape, power, left):
    """Values that a row does not attend, behind it or left of its window, 2^power times the others: its bits stay."""
    heads, kvh, hd, kv, new = shape
    window = new // 3 + 1 if left else 0
    p = Pool(np.random.default_rng(44), [kv], kvh, hd, 64, typ).fill()
    half = new // 2
    a = p.attend([new], heads, max_q=new, window=window)
    if left:  # rows from `half` on attend nothing at or in front of half's position less the window
        keep, swap = slice(half, None), slice(0, kv - new + half - window + 1)
    else:
        keep, swap = slice(0, half), slice(kv - new + half, None)
    p.v[0][swap] *= np.float32(2.0 ** power)
    p.fill()
    b = p.attend([new], heads, max_q=new, window=window, q=p.q)
    close(b, p, new, 1 / np.sqrt(hd), window, keep)
    assert np.array_equal(a[keep], b[keep]), f"{(a[keep] != b[keep]).sum()} values changed"
    close(b, p, new, 1 / np.sqrt(hd), window)


def test_in_place_at_another_stride_is_refused():
    """out = q needs q's stride: rows written at another one would be queries that other blocks still read."""
    p = pool(45, "q8", ROW[1])
    L, x = wv.lib(), torch.zeros(1 << 16, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    b = KVBatch(1, 9, 1, i.data_ptr(), i.data_ptr(), i.data_ptr())

    def call(qs, os, out):
        return L.wv_kv_attention_dev(p.kv.handle, 0, ctypes.byref(b), x.data_ptr(), qs, 8, 1.0, 0, out, os, None, 0, None)
    assert call(1025, 0, x.data_ptr()) == -2 and b"out is q" in L.wv_last_error()
    assert call(0, 2048, x.data_ptr()) == -2
    assert call(1024, 0, x.data_ptr()) == 0 and call(1025, 0, x.data_ptr() + 4 * 16384) == 0
    wv.sync()


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("n", [5, 1024])  # row by row, and tiles of 32 rows
def test_the_largest_rows_read_back_finite(typ, n):
    """Rows up to f32's largest value: a code times its scale never rounds to infinity. In between the codes are the
    nearest ones: half a step of an 11-bit fp16 code or of 1 / 127, a whole one at the very end."""
    rng, big = np.random.default_rng(46), np.finfo(np.float32).max
    x = (rng.uniform(-1, 1, (n, 8, 64)) * big).astype(np.float32)
    x[:, :, 0] = np.float32(big) * np.where(rng.random((n, 8)) < 0.5, -1, 1)
    x[1, :, 1] = np.float32(3.4021e38)
    kv = KVCache(1, 8, 64, 32, n // 32 + 1, typ)
    dx, ds = dev(x), dev(np.arange(n), np.int64)
    k, v = (torch.zeros(n, 8, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    kv.write_dev(0, dx.data_ptr(), dx.data_ptr(), ds.data_ptr(), n)
    kv.read_dev(0, ds.data_ptr(), n, k.data_ptr(), v.data_ptr())
    wv.sync()
    for got in (k, v):
        off = np.abs(got.cpu().numpy().astype(np.float64) - x) / np.float64(big)
        assert off.max() <= (2.0 ** -11 if typ == "f16" else 0.5 / 127 + 2.0 ** -23)
