"""The paged KV cache on the device: rows written and read back bit by bit
against their definition, and the attention of new tokens against float64
(kv_ref), at the sizes, strides, pages and masks where either can go wrong."""
import ctypes
import math

import numpy as np
import pytest
import torch

import welvet_amd as wv
from kv_ref import attention, stored
from welvet_amd.kv import KVBatch, KVCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def dev(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x if dtype is None else np.asarray(x, dtype))).cuda()


def rows(rng, n, heads, hd, outliers=False):
    x = rng.standard_normal((n, heads, hd)).astype(np.float32)
    if outliers:
        x[..., rng.permutation(hd)[:3]] *= 7
    return x


class Pool:
    """A cache of one layer (of `layers`), sequences on shuffled pages of it, and what it should hold."""

    def __init__(self, rng, lens, kv_heads, hd, page, typ, layers=1, layer=0, extra=2):
        self.rng, self.typ, self.page, self.layer, self.hd, self.kv_heads = rng, typ, page, layer, hd, kv_heads
        self.width = max(1, max(-(-n // page) for n in lens))
        n_pages = len(lens) * self.width + extra
        self.kv = KVCache(layers, kv_heads, hd, page, n_pages, typ)
        self.table = rng.permutation(n_pages)[: len(lens) * self.width].reshape(len(lens), self.width).astype(np.int32)
        self.lens = lens
        self.k = [rows(rng, n, kv_heads, hd, True) for n in lens]
        self.v = [rows(rng, n, kv_heads, hd) for n in lens]

    def slots(self, b):
        j = np.arange(self.lens[b])
        return self.table[b][j // self.page].astype(np.int64) * self.page + j % self.page

    def fill(self):
        k, v = np.concatenate(self.k), np.concatenate(self.v)
        sl = np.concatenate([self.slots(b) for b in range(len(self.lens))])
        dk, dv, ds = dev(k), dev(v), dev(sl)
        torch.cuda.synchronize()
        self.kv.write_dev(self.layer, dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), len(sl))
        wv.sync()
        return self

    def attend(self, new, heads, scale=None, window=0, max_q=0, q=None, pad=0, stream=None, table=None, kv_len=None):
        """Rows out [sum(new) + pad, heads, hd]; padding rows start as 7."""
        scale = 1.0 / math.sqrt(self.hd) if scale is None else scale
        nt = sum(new) + pad
        self.q = rows(self.rng, nt, heads, self.hd) if q is None else q
        dq = dev(self.q)
        out = torch.full((nt, heads, self.hd), 7.0, device="cuda")
        cu = dev(np.concatenate([[0], np.cumsum(new)]), np.int32)
        ln = dev(self.lens if kv_len is None else kv_len, np.int32)
        tb = dev(self.table if table is None else table)
        torch.cuda.synchronize()
        b = KVBatch(len(new), nt, tb.shape[1], cu.data_ptr(), ln.data_ptr(), tb.data_ptr(), max_q=max_q)
        self.kv.attention_dev(self.layer, b, dq.data_ptr(), out.data_ptr(), heads, scale, window, stream=stream)
        wv.sync(stream)
        return out.cpu().numpy()

    def check(self, out, new, scale=None, window=0, present=None, lens=None):
        scale = 1.0 / math.sqrt(self.hd) if scale is None else scale
        at = 0
        for b, n in enumerate(new):
            m = self.lens[b] if lens is None else lens[b]
            pr = None if present is None else present[b][:m]
            ref, tol = attention(self.q[at:at + n], stored(self.k[b], self.typ)[:m], stored(self.v[b], self.typ)[:m],
                                 n, np.float32(scale), window, pr)
            got = out[at:at + n].astype(np.float64)
            assert np.array_equal(np.isnan(got), np.isnan(ref)), f"sequence {b}"
            bad = np.abs(got - ref) > tol
            assert not bad.any(), f"sequence {b}: off by {np.nanmax(np.abs(got - ref))}, {bad.sum()} values"
            at += n
        assert (out[at:] == 7.0).all(), "padding rows written"


# ------------------------------------------------------------ write and read

@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("hd,kv_heads,page,n", [(128, 8, 32, 1), (64, 1, 32, 5), (128, 3, 64, 77), (64, 8, 256, 300),
                                                (128, 2, 128, 129)])
def test_write_read_exact(typ, hd, kv_heads, page, n):
    rng = np.random.default_rng(n + hd)
    p = Pool(rng, [n], kv_heads, hd, page, typ, layers=3, layer=1).fill()
    sl = dev(p.slots(0))
    k, v = (torch.full((n, kv_heads, hd), 9.0, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    p.kv.read_dev(1, sl.data_ptr(), n, k.data_ptr(), v.data_ptr())
    wv.sync()
    assert np.array_equal(k.cpu().numpy(), stored(p.k[0], typ))
    assert np.array_equal(v.cpu().numpy(), stored(p.v[0], typ))
    for layer in (0, 2):  # the other layers were left alone
        p.kv.read_dev(layer, sl.data_ptr(), n, k.data_ptr(), v.data_ptr())
        wv.sync()
        assert not k.cpu().numpy().any() and not v.cpu().numpy().any()


@pytest.mark.parametrize("typ", ["f16", "q8"])
def test_write_read_special_rows(typ):
    """Zeros, ties, tiny and huge rows, NaN and infinity, half-way quotients; skipped and foreign slots."""
    hd, kvh = 64, 2
    rng = np.random.default_rng(3)
    x = rows(rng, 12, kvh, hd)
    x[0] = 0
    x[1] *= np.float32(1e-32)          # below 2^-100: held as zeros
    x[2] *= np.float32(1e30)
    x[3, 0, 5], x[4, 1, 9] = np.nan, -np.inf
    x[5, 0, :] = np.float32(127) * np.sign(x[5, 0, :])
    x[5, 0, 1:] = (np.arange(63) - 31.5).astype(np.float32)  # quotients k + 0.5 with a scale of 1
    x[5, 0, 0] = 127
    x[6] = -x[6]
    x[7, :, :] = np.float32(3.4e38) * np.sign(x[7])
    x[8] *= np.float32(2.0 ** -99)
    x[9, :, 1:] = 0                    # one value alone
    slots = np.arange(12, dtype=np.int64) * 5
    slots[10], slots[11] = -1, 32 * 4  # padding, and the first position past the pool
    kv = KVCache(1, kvh, hd, 32, 4, typ)
    dk, dv, ds = dev(x), dev(x[::-1]), dev(slots)
    torch.cuda.synchronize()
    kv.write_dev(0, dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), 12)
    k, v = (torch.full((128 + 2, kvh, hd), 9.0, device="cuda") for _ in range(2))
    every = dev(np.concatenate([np.arange(128), [-7, 1 << 40]]), np.int64)
    torch.cuda.synchronize()
    kv.read_dev(0, every.data_ptr(), 130, k.data_ptr(), v.data_ptr())
    wv.sync()
    want_k, want_v = np.zeros((130, kvh, hd)), np.zeros((130, kvh, hd))
    want_k[slots[:10]], want_v[slots[:10]] = stored(x, typ)[:10], stored(x[::-1], typ)[:10]
    assert np.array_equal(k.cpu().numpy(), want_k, equal_nan=True)
    assert np.array_equal(v.cpu().numpy(), want_v, equal_nan=True)
    # a finite row over a NaN one: nothing of it stays
    ds2 = dev(slots[3:4])
    torch.cuda.synchronize()
    kv.write_dev(0, dk[6:].data_ptr(), dv[6:].data_ptr(), ds2.data_ptr(), 1)
    kv.read_dev(0, ds2.data_ptr(), 1, k.data_ptr(), v.data_ptr())
    wv.sync()
    assert np.array_equal(k[0].cpu().numpy(), stored(x[6], typ))


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("stride_k,stride_v,off", [(131, 128, 0), (160, 133, 1), (128, 128, 2)])
def test_write_read_strides(typ, stride_k, stride_v, off):
    """Rows inside wider ones, at odd strides and addresses; what lies between them stays."""
    hd, kvh, n = 64, 2, 37
    rng = np.random.default_rng(stride_k)
    big_k, big_v = (rng.standard_normal(off + n * s + 8).astype(np.float32) for s in (stride_k, stride_v))
    take = [np.stack([b[off + t * s: off + t * s + kvh * hd] for t in range(n)]).reshape(n, kvh, hd)
            for b, s in ((big_k, stride_k), (big_v, stride_v))]
    kv = KVCache(1, kvh, hd, 64, 2, typ)
    slots = rng.permutation(128)[:n].astype(np.int64)
    dk, dv, ds = dev(big_k), dev(big_v), dev(slots)
    torch.cuda.synchronize()
    kv.write_dev(0, dk.data_ptr() + 4 * off, dv.data_ptr() + 4 * off, ds.data_ptr(), n, stride_k, stride_v)
    ok, ov = torch.full_like(dk, 9.0), torch.full_like(dv, 9.0)
    torch.cuda.synchronize()
    kv.read_dev(0, ds.data_ptr(), n, ok.data_ptr() + 4 * off, ov.data_ptr() + 4 * off, stride_k, stride_v)
    wv.sync()
    for out, x, s in ((ok, take[0], stride_k), (ov, take[1], stride_v)):
        want = np.full(out.numel(), 9.0, np.float32)
        for t in range(n):
            want[off + t * s: off + t * s + kvh * hd] = stored(x[t], typ).ravel()
        assert np.array_equal(out.cpu().numpy(), want)


def slot_order(kind, rng, n, pool):
    """n different slots of the pool in some order, -1 and others outside it among them."""
    if kind == "shifted":  # runs that begin inside a block and inside a word of four keys
        cut = [0, 1, 6, 39, 104, n]
        at = [3, 65, 130, 195, 322, 420]
        return np.concatenate([np.arange(a, a + j - i) for a, i, j in zip(at, cut, cut[1:])])
    if kind == "holes":    # every seventh row is padding
        s = np.arange(5, 5 + n)
        s[::7] = np.where(np.arange(len(s[::7])) % 2, -1, pool + np.arange(len(s[::7])) % 9)
        return s
    if kind == "falling":
        return np.arange(pool - 1, pool - 1 - n, -1)
    if kind == "words":    # words of four whole, in any order
        return (rng.permutation(pool // 4)[:-(-n // 4), None] * 4 + np.arange(4)).ravel()[:n]
    return rng.permutation(pool)[:n]


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("kind", ["shifted", "holes", "falling", "words", "any"])
@pytest.mark.parametrize("kv_heads,hd,page,n,odd", [(41, 64, 32, 401, 0), (36, 128, 64, 500, 3), (64, 128, 256, 256, 0)])
def test_write_read_many_rows(typ, kind, kv_heads, hd, page, n, odd):
    """Enough rows for whole tiles of them; what no slot names stays."""
    rng = np.random.default_rng(n)
    pool = 1024
    slots = np.asarray(slot_order(kind, rng, n, pool), np.int64)
    w = kv_heads * hd + odd
    x = [rows(rng, 1, n, w)[0] for _ in range(2)]
    x[0][7, 3], x[1][40, 1], x[1][90] = np.nan, np.inf, 0
    kv = KVCache(1, kv_heads, hd, page, pool // page, typ)
    base = rows(rng, pool, kv_heads, hd)
    every = np.arange(pool, dtype=np.int64)
    db, de, dk, dv, ds = dev(base), dev(every), dev(x[0]), dev(x[1]), dev(slots)
    torch.cuda.synchronize()
    kv.write_dev(0, db.data_ptr(), db.data_ptr(), de.data_ptr(), pool)
    kv.write_dev(0, dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), n, w, w)
    inside = (slots >= 0) & (slots < pool)
    for order in (every, slots):
        m = len(order)
        out = [torch.full((m + 1, w), 9.0, device="cuda") for _ in range(2)]
        do = dev(order)
        torch.cuda.synchronize()
        kv.read_dev(0, do.data_ptr(), m, out[0].data_ptr(), out[1].data_ptr(), w, w)
        wv.sync()
        for o, rows_in in zip(out, x):
            cache = stored(base, typ)
            cache[slots[inside]] = stored(rows_in[inside][:, :kv_heads * hd].reshape(-1, kv_heads, hd), typ)
            want = np.full((m + 1, w), 9.0, np.float32)
            ok = (order >= 0) & (order < pool)
            want[:m, :kv_heads * hd] = np.where(ok[:, None], cache[np.where(ok, order, 0)].reshape(m, -1), 0)
            assert np.array_equal(o.cpu().numpy(), want, equal_nan=True)


# ----------------------------------------------------------------- attention

LAYOUTS = [(8, 8, 64), (8, 2, 128), (5, 1, 64), (32, 8, 128), (6, 2, 64), (24, 1, 128)]


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("kv,new", [(1, 1), (31, 1), (33, 3), (200, 7), (65, 65), (700, 130), (2500, 301)])
def test_attention_one_sequence(typ, heads, kv_heads, hd, kv, new):
    rng = np.random.default_rng(kv * 7 + heads)
    p = Pool(rng, [kv], kv_heads, hd, 32, typ).fill()
    p.check(p.attend([new], heads), [new])


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 50, 4096])
def test_attention_ragged_batch(typ, page, window):
    """Chunks beside single tokens, an idle sequence, one with no keys at all, padding rows behind the last."""
    rng = np.random.default_rng(page + window)
    lens, new = [300, 1, 97, 64, 513, 40], [20, 1, 1, 0, 150, 40]
    p = Pool(rng, lens, 2, 64, page, typ, layers=2, layer=1).fill()
    for max_q in (0, 150, 1):  # a wrong hint costs time only
        p.check(p.attend(new, 6, window=window, max_q=max_q, pad=3), new, window=window)


def test_attention_rows_without_keys():
    """kv_len under the new tokens' count, and 0: those rows are zeros."""
    rng = np.random.default_rng(1)
    p = Pool(rng, [64, 64], 2, 64, 32, "q8").fill()
    out = p.attend([5, 4], 4, kv_len=[3, 0])
    ref, tol = attention(p.q[2:5], stored(p.k[0], "q8")[:3], stored(p.v[0], "q8")[:3], 3, np.float32(0.125))
    assert not out[:2].any() and not out[5:].any()
    assert (np.abs(out[2:5] - ref) <= tol).all()


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("new", [1, 90])
def test_attention_absent_pages(typ, new):
    """Pages outside the pool hold no keys; a table narrower than kv_len ends the keys."""
    rng = np.random.default_rng(new)
    p = Pool(rng, [400], 2, 64, 64, typ).fill()
    table = p.table.copy()
    table[0, 1], table[0, 4] = -1, 1 << 30
    present = np.ones(400, bool)
    present[64:128] = present[256:320] = False
    p.check(p.attend([new], 8, table=table), [new], present=[present])
    present[:] = True
    present[320:] = False
    p.check(p.attend([new], 8, table=p.table[:, :5]), [new], present=[present])


@pytest.mark.parametrize("typ", ["f16", "q8"])
def test_attention_nan_where_masked(typ):
    """NaN rows that no query sees change nothing: future tokens, positions behind the keys, left of the window."""
    rng = np.random.default_rng(5)
    p = Pool(rng, [160], 2, 64, 32, typ)
    clean_k, clean_v = p.k[0].copy(), p.v[0].copy()
    p.k[0][150:] = np.nan
    p.v[0][150:] = np.inf
    p.k[0][:40], p.v[0][:40] = np.inf, np.nan
    p.fill()
    out = p.attend([30], 4, window=60, kv_len=[150])
    p.k[0], p.v[0] = clean_k, clean_v
    p.check(out, [30], window=60, lens=[150])
    # and what does attend to one is NaN, that row alone
    p.k[0][140] = np.nan
    p.fill()
    out = p.attend([30], 4, kv_len=[150])
    assert np.isnan(out[20:]).all() and np.isfinite(out[:20]).all()


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("size", [1e-25, 1e-3, 1e4, 1e25])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_magnitudes(typ, size, new):
    """V of any magnitude, a few rows far above the others; queries and keys whose product is ordinary."""
    rng = np.random.default_rng(9)
    p = Pool(rng, [300], 2, 128, 32, typ)
    p.v[0] *= np.float32(size)
    p.v[0][::37] *= np.float32(300)
    p.k[0] *= np.float32(1 / size if size < 1 else size)
    p.fill()
    q = rows(rng, new, 8, 128) * np.float32(size if size < 1 else 1 / size)
    p.check(p.attend([new], 8, q=q), [new])


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("new", [1, 33])
def test_attention_large_scores(typ, new):
    """Scores of hundreds: one key takes all, running maxima grow by as much."""
    rng = np.random.default_rng(10)
    p = Pool(rng, [515], 1, 64, 64, typ)
    p.k[0] *= np.float32(40) * np.linspace(0.1, 1, 515).astype(np.float32)[:, None, None]
    p.fill()
    p.check(p.attend([new], 4), [new])


def test_attention_long_split_and_deterministic():
    """A long cache cut into ranges: against float64, and the same bits again; also with the caller's scratch."""
    rng = np.random.default_rng(11)
    p = Pool(rng, [9001], 1, 128, 64, "q8").fill()
    a = p.attend([1], 4)
    p.check(a, [1])
    assert np.array_equal(a, p.attend([1], 4, q=p.q))
    b = KVBatch(1, 1, p.width, 0, 0, 0)
    assert p.kv.attention_scratch(b, 4) > 0


# The kernel for many rows takes long chunks: these shapes, of whatever type.

@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv_heads,hd,kv,new", [(32, 8, 64, 2100, 2048), (64, 16, 128, 1100, 1024),
                                                      (24, 24, 64, 2750, 2747), (32, 8, 128, 4200, 515),
                                                      (24, 4, 128, 9001, 203), (64, 16, 64, 1900, 1900)])
def test_many_rows_one_sequence(typ, heads, kv_heads, hd, kv, new):
    """Whole prompts, a chunk behind cached keys, one cut into key ranges (515 tokens over 4200 keys)."""
    rng = np.random.default_rng(kv + heads)
    p = Pool(rng, [kv], kv_heads, hd, 64, typ).fill()
    a = p.attend([new], heads, max_q=new)
    p.check(a, [new])
    assert np.array_equal(a, p.attend([new], heads, max_q=new, q=p.q))


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("window", [0, 200])
def test_many_rows_ragged_batch(typ, window):
    """Long chunks beside single tokens and an idle sequence, padding rows, pages outside the pool."""
    rng = np.random.default_rng(window + 21)
    lens, new = [1500, 700, 64, 1000, 333, 3], [1100, 0, 1, 1000, 300, 2]
    p = Pool(rng, lens, 8, 64, 32, typ, layers=2, layer=1).fill()
    p.check(p.attend(new, 32, window=window, pad=5), new, window=window)
    table = p.table.copy()
    table[0, 3], table[3, 7], table[3, 31] = -1, 1 << 30, len(lens) * p.width + 2
    present = [np.ones(n, bool) for n in lens]
    present[0][96:128] = present[3][224:256] = present[3][992:] = False
    p.check(p.attend(new, 32, window=window, table=table, max_q=1100), new, window=window, present=present)


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("new", [6, 1900])
def test_more_tokens_than_keys_and_short_tables(typ, new):
    """A sequence whose first tokens stand in front of the keys, and one whose table ends before its keys do."""
    rng = np.random.default_rng(new)
    p = Pool(rng, [max(new // 2, 3)], 16, 64, 64, typ).fill()
    out = p.attend([new], 64, max_q=new)
    p.check(out, [new])
    assert not out[:new - p.lens[0]].any()
    p = Pool(rng, [new + 200], 16, 64, 64, typ).fill()
    cut = (new + 150) // 64
    present = [np.arange(new + 200) < 64 * cut]
    p.check(p.attend([new], 64, max_q=new, table=p.table[:, :cut].copy()), [new], present=present)


@pytest.mark.parametrize("typ", ["f16", "q8"])
def test_many_rows_nan_and_magnitudes(typ):
    """NaN rows behind the keys and left of the window change nothing, a NaN key the rows that attend to it;
    V rows far above and below the others, scores of hundreds."""
    rng = np.random.default_rng(31)
    p = Pool(rng, [2200], 8, 64, 32, typ)
    p.v[0][::41] *= np.float32(1e4)
    p.v[0][7::53] *= np.float32(1e-6)
    p.k[0][:, ::2] *= np.float32(30)
    clean = p.k[0].copy(), p.v[0].copy()
    p.k[0][2100:], p.v[0][2100:] = np.nan, np.inf
    p.k[0][:20], p.v[0][:20] = np.inf, np.nan
    p.fill()
    out = p.attend([2048], 32, window=30, kv_len=[2100])
    p.k[0], p.v[0] = clean
    p.check(out, [2048], window=30, lens=[2100])
    p.k[0][2090, 3], p.v[0][2095, 5] = np.nan, np.nan
    p.fill()
    out = p.attend([2048], 32, kv_len=[2100])
    bad = np.isnan(out)
    want = np.zeros_like(bad)
    want[2090 - 52:, 12:16] = want[2095 - 52:, 20:24] = True
    assert np.array_equal(bad, want)


def test_attention_strides_and_in_place():
    rng = np.random.default_rng(12)
    p = Pool(rng, [130], 2, 64, 32, "f16").fill()
    big = rng.standard_normal((9, 4 * 64 + 33)).astype(np.float32)
    p.q = np.ascontiguousarray(big[:, :256]).reshape(9, 4, 64)
    dq = dev(big)
    cu, ln, tb = dev([0, 9], np.int32), dev([130], np.int32), dev(p.table)
    torch.cuda.synchronize()
    b = KVBatch(1, 9, p.width, cu.data_ptr(), ln.data_ptr(), tb.data_ptr())
    p.kv.attention_dev(0, b, dq.data_ptr(), dq.data_ptr(), 4, 0.125, q_stride=289, out_stride=289)
    wv.sync()
    got = dq.cpu().numpy()
    p.check(got[:, :256].reshape(9, 4, 64).copy(), [9], scale=0.125)
    assert np.array_equal(got[:, 256:], big[:, 256:])


@pytest.mark.parametrize("scratch", [False, True])
def test_attention_graph_replays(scratch):
    """Write and attend captured; each replay takes the lengths, tables and rows that then lie in the arrays."""
    rng = np.random.default_rng(13)
    p = Pool(rng, [2000], 2, 64, 32, "q8").fill()
    st = torch.cuda.Stream()
    q, out = torch.zeros(1, 8, 64, device="cuda"), torch.zeros(1, 8, 64, device="cuda")
    cu, ln, tb = dev([0, 1], np.int32), dev([2000], np.int32), dev(p.table)
    nk, nv, sl = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda"), dev([0], np.int64)
    b = KVBatch(1, 1, p.width, cu.data_ptr(), ln.data_ptr(), tb.data_ptr(), max_q=1)
    buf = torch.zeros(max(1, p.kv.attention_scratch(b, 8)), dtype=torch.uint8, device="cuda")
    assert buf.numel() > 1
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        h = st.cuda_stream
        p.kv.write_dev(0, nk.data_ptr(), nv.data_ptr(), sl.data_ptr(), 1, stream=h)
        p.kv.attention_dev(0, b, q.data_ptr(), out.data_ptr(), 8, 0.125, stream=h,
                           scratch_ptr=buf.data_ptr() if scratch else None,
                           scratch_bytes=buf.numel() if scratch else 0)
    for i, length in enumerate((2000, 17, 1500, 2000)):
        x = [rows(rng, 1, h, 64) for h in (8, 2, 2)]
        for t, y in zip((q, nk, nv), x):
            t.copy_(torch.from_numpy(y))
        ln.fill_(length)
        sl.fill_(int(p.slots(0)[length - 1]))
        p.q, p.k[0][length - 1], p.v[0][length - 1] = x[0], x[1][0], x[2][0]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        p.check(out.cpu().numpy(), [1], scale=0.125, lens=[length])
        eager = p.attend([1], 8, scale=0.125, q=p.q, kv_len=[length])  # eager work between the replays
        p.check(eager, [1], scale=0.125, lens=[length])


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("max_q", [0, 1])
def test_attention_one_chunk_among_tokens(typ, max_q):
    """Many single tokens, idle sequences, and one or two chunks that the batch's average (or a max_q too small)
    does not let expect."""
    rng = np.random.default_rng(max_q + 77)
    new = [1] * 30 + [0, 100, 1, 0, 0, 37] + [1] * 25
    lens = [int(n) for n in rng.integers(1, 300, len(new))]
    lens[31], lens[35] = 250, 37
    p = Pool(rng, lens, 2, 64, 32, typ).fill()
    p.check(p.attend(new, 4, max_q=max_q, pad=3), new)


@pytest.mark.parametrize("new", [3, 600])
def test_attention_of_zero_queries(new):
    """Queries of zeros and a scale that underflows: the plain mean of the values, the masked keys left out."""
    p = Pool(np.random.default_rng(new), [700], 2, 64, 32, "f16").fill()
    q = np.zeros((new, 8, 64), np.float32)
    out = p.attend([new], 8, scale=1e-12, q=q, max_q=new)
    p.check(out, [new], scale=1e-12)
    assert np.isfinite(out).all()


def test_attention_two_streams():
    """Split calls on two streams at once do not share partials."""
    rng = np.random.default_rng(14)
    p = Pool(rng, [5000, 4000], 1, 64, 64, "f16").fill()
    calls = []
    for b in range(2):
        st = torch.cuda.Stream()
        q = rows(rng, 1, 4, 64)
        calls.append([st, q, dev(q), torch.zeros(8, 1, 4, 64, device="cuda"), dev([0, 1], np.int32),
                      dev([p.lens[b]], np.int32), dev(p.table[b:b + 1])])
    torch.cuda.synchronize()
    for i in range(8):
        for st, _, dq, out, cu, ln, tb in calls:
            kb = KVBatch(1, 1, p.width, cu.data_ptr(), ln.data_ptr(), tb.data_ptr())
            p.kv.attention_dev(0, kb, dq.data_ptr(), out[i].data_ptr(), 4, 0.125, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for b, (_, q, _, out, *_rest) in enumerate(calls):
        ref, tol = attention(q, stored(p.k[b], "f16"), stored(p.v[b], "f16"), 1, np.float32(0.125))
        for i in range(8):
            assert (np.abs(out[i].cpu().numpy() - ref) <= tol).all()


def test_refusals_with_a_cache():
    kv = KVCache(2, 2, 64, 32, 4, "q8")
    L = wv.lib()
    x = torch.zeros(4096, device="cuda")
    i = torch.zeros(64, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    P, I = x.data_ptr(), i.data_ptr()
    assert L.wv_kv_write_dev(kv.handle, 2, P, P, 0, 0, I, 1, None) == -1
    assert L.wv_kv_write_dev(kv.handle, -1, P, P, 0, 0, I, 1, None) == -1
    assert L.wv_kv_write_dev(kv.handle, 0, P, P, 0, 0, I, -1, None) == -2
    assert L.wv_kv_write_dev(kv.handle, 0, P, P, 127, 0, I, 1, None) == -2
    assert L.wv_kv_write_dev(kv.handle, 0, P, P, 0, 0, I, (1 << 27) + 1, None) == -2
    assert L.wv_kv_read_dev(kv.handle, 0, I, (1 << 27) + 1, P, P, 0, 0, None) == -2
    assert L.wv_kv_write_dev(kv.handle, 0, None, P, 0, 0, I, 1, None) == -1
    assert L.wv_kv_read_dev(kv.handle, 0, None, 1, P, P, 0, 0, None) == -1
    assert L.wv_kv_write_dev(kv.handle, 0, None, None, 0, 0, None, 0, None) == 0
    assert L.wv_kv_read_dev(kv.handle, 0, None, 0, None, None, 0, 0, None) == 0

    def attn(b=None, layer=0, q=P, heads=4, scale=1.0, window=0, qs=0, scratch=None, sb=0):
        b = KVBatch(1, 1, 1, I, I, I) if b is None else b
        return L.wv_kv_attention_dev(kv.handle, layer, ctypes.byref(b), q, qs, heads, scale, window, P, 0, scratch, sb,
                                     None)
    assert attn(layer=2) == -1 and attn(heads=3) == -2 and attn(heads=0) == -2
    assert attn(scale=0.0) == -1 and attn(scale=float("nan")) == -1 and attn(scale=float("inf")) == -1
    assert attn(window=-1) == -2 and attn(qs=255) == -2 and attn(q=None) == -1
    assert attn(KVBatch(-1, 1, 1, I, I, I)) == -2 and attn(KVBatch(1, -1, 1, I, I, I)) == -2
    assert attn(KVBatch(1, 1, 1 << 26, I, I, I)) == -2 and attn(KVBatch(1, 1 << 30, 1, I, I, I)) == -2
    assert attn(KVBatch(1, 1, 1, None, I, I)) == -1 and attn(KVBatch(1, 1, 1, I, I, None)) == -1
    assert attn(KVBatch(0, 5, 1, None, None, None)) == 0 and attn(KVBatch(3, 0, 1, None, None, None)) == 0
    assert attn(KVBatch(1, 1, 64, I, I, I), scratch=P, sb=16) == -2
    assert attn(KVBatch(1, 1, 64, I, I, I), scratch=P + 4, sb=1 << 20) == -1
    assert kv.info()["device_bytes"] == 2 * (2 * 128 * 2 * 64 + 128 * 2 * 8)
    kv.free()
    assert L.wv_kv_free(12345678) == -7
