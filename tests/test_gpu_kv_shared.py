"""Attention of batches whose sequences share their first keys, against every
sequence's own attention in float64 (kv_ref)."""
import math

import numpy as np
import pytest
import torch

import welvet_amd as wv
from kv_ref import attention, stored
from welvet_amd.kv import KVBatch, KVCache, KVGroups

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def dev(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x if dtype is None else np.asarray(x, dtype))).cuda()


WIDE = 65536  # positions of a crowd's table


class Batch:
    """Groups of sequences in a cache: `groups` lists (members, shared), the first `before` sequences are of no group,
    nor are those behind the last; lens and new per sequence. Members hold the pages of the prefix that are full in
    common. crowd: 64 short sequences more, as a last group, and a table so wide that attention over whole sequences
    would take longest: shared keys are read once for their group then, else where a call is large enough for that."""

    def __init__(self, rng, groups, lens, new, kv_heads, hd, page, typ, before=0, pad=0, layers=1, layer=0,
                 crowd=False):
        if crowd:
            at = before + sum(m for m, _ in groups)
            groups = list(groups) + [(64, 64)]
            lens = list(lens[:at]) + [65 + i % 5 for i in range(64)] + list(lens[at:])
            new = list(new[:at]) + [1] * 64 + list(new[at:])
        self.crowd = crowd
        self.rng, self.lens, self.new, self.typ, self.page, self.hd = rng, lens, new, typ, page, hd
        self.kv_heads, self.layer, self.pad, self.n_groups = kv_heads, layer, pad, len(groups)
        members = [m for m, _ in groups]
        self.group_cu = np.concatenate([[0], np.cumsum(members)]) + before
        self.shared = [s for _, s in groups]
        held = [-(-n // page) for n in lens]
        width = WIDE // page if crowd else max(max(held), 1)
        pool = sum(held) + 3
        free = list(rng.permutation(pool))
        self.table = np.full((len(lens), width), -1, np.int32)
        self.k, self.v = [], []
        self.fresh = []
        for b, n in enumerate(lens):
            k, v = (rng.standard_normal((n, kv_heads, hd)).astype(np.float32) for _ in range(2))
            k[..., rng.permutation(hd)[:3]] *= 5
            g = int(np.searchsorted(self.group_cu, b, side="right")) - 1
            lead = int(self.group_cu[g]) if 0 <= g < len(groups) else b
            common = 0
            if lead != b:
                s = min(self.shared[g], n, lens[lead])
                k[:s], v[:s] = self.k[lead][:s], self.v[lead][:s]
                common = s // page
                self.table[b, :common] = self.table[lead, :common]
            self.table[b, common:held[b]] = [free.pop() for _ in range(held[b] - common)]
            self.fresh.append(common * page)
            self.k.append(k)
            self.v.append(v)
        self.kv = KVCache(layers, kv_heads, hd, page, pool, typ)
        self.fill()

    def fill(self):
        k, v, sl = [], [], []
        for b, n in enumerate(self.lens):
            j = np.arange(self.fresh[b], n)
            sl.append(self.table[b][j // self.page].astype(np.int64) * self.page + j % self.page)
            k.append(self.k[b][self.fresh[b]:])
            v.append(self.v[b][self.fresh[b]:])
        dk, dv, ds = dev(np.concatenate(k)), dev(np.concatenate(v)), dev(np.concatenate(sl))
        torch.cuda.synchronize()
        self.kv.write_dev(self.layer, dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), ds.numel())
        wv.sync()

    def arrays(self, heads):
        nt = sum(self.new) + self.pad
        self.q = self.rng.standard_normal((nt, heads, self.hd)).astype(np.float32)
        self.d = [dev(np.concatenate([[0], np.cumsum(self.new)]), np.int32), dev(self.lens, np.int32), dev(self.table),
                  dev(self.group_cu, np.int32), dev(self.shared, np.int32), dev(self.q)]
        self.out = torch.full((nt, heads, self.hd), 7.0, device="cuda")
        torch.cuda.synchronize()

    def structs(self, max_q=0, max_shared=0):
        cu, ln, tb, gc, sh, _ = self.d
        b = KVBatch(len(self.new), self.out.shape[0], tb.shape[1], cu.data_ptr(), ln.data_ptr(), tb.data_ptr(), max_q)
        return b, KVGroups(self.n_groups, gc.data_ptr(), sh.data_ptr(), max_shared)

    def attend(self, heads, window=0, max_q=0, max_shared=0, in_place=False, grouped=None, **kw):
        self.arrays(heads)
        b, g = self.structs(max_q, max_shared)
        if self.crowd and max_shared == window == 0 and grouped is None or grouped:  # shared and own keys' partial rows
            assert self.kv.attention_shared_scratch(b, g, heads, window) != self.kv.attention_scratch(b, heads, window)
        q = self.d[5]
        out = q if in_place else self.out
        self.kv.attention_shared_dev(self.layer, *self.structs(max_q, max_shared), q.data_ptr(), out.data_ptr(), heads,
                                     1.0 / math.sqrt(self.hd), window, **kw)
        wv.sync(kw.get("stream"))
        return out.cpu().numpy()

    def again(self, heads, max_q, max_shared):
        out = torch.zeros_like(self.out)
        torch.cuda.synchronize()
        self.kv.attention_shared_dev(self.layer, *self.structs(max_q, max_shared), self.d[5].data_ptr(), out.data_ptr(),
                                     heads, 1.0 / math.sqrt(self.hd))
        wv.sync()
        return out.cpu().numpy()

    def check(self, out, window=0, present=None, padding=True):
        at = 0
        for b, n in enumerate(self.new):
            ref, tol = attention(self.q[at:at + n], stored(self.k[b], self.typ), stored(self.v[b], self.typ), n,
                                 np.float32(1.0 / math.sqrt(self.hd)), window, None if present is None else present[b])
            got = out[at:at + n].astype(np.float64)
            assert np.array_equal(np.isnan(got), np.isnan(ref)), f"sequence {b}"
            bad = np.abs(got - ref) > tol
            assert not bad.any(), f"sequence {b}: off by {np.nanmax(np.abs(got - ref))}, {bad.sum()} values"
            at += n
        if padding:
            assert (out[at:] == 7.0).all(), "padding rows written"


@pytest.mark.parametrize("crowd", [False, True])
@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("shared", [0, 1, 31, 32, 33, 64, 95, 500])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 128, 32), (3, 3, 64, 64), (16, 2, 64, 32)])
def test_one_group(typ, shared, heads, kv_heads, hd, page, crowd):
    rng = np.random.default_rng(shared + hd)
    new = [1, 1, 3, 0, 2]
    lens = [shared + n + x for n, x in zip(new, (0, 1, 40, 7, 130))]
    b = Batch(rng, [(5, shared)], lens, new, kv_heads, hd, page, typ, pad=2, crowd=crowd)
    b.check(b.attend(heads))
    b.check(b.attend(heads, max_q=3, max_shared=shared))


@pytest.mark.parametrize("crowd", [False, True])
@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("window", [0, 1, 50, 400])
@pytest.mark.parametrize("hint", [0, 1, 600, 100000])
def test_several_groups(typ, window, hint, crowd):
    """Groups of several sizes, an empty one and one of one sequence, sequences before and behind them, windows;
    whatever the launch is told."""
    rng = np.random.default_rng(window + hint)
    groups = [(4, 300), (0, 64), (1, 200), (3, 5), (6, 601)]
    before, after = 2, 3
    lead = [0] * before + [s for m, s in groups for _ in range(m)] + [0] * after
    new = [int(x) for x in rng.integers(0, 5, len(lead))]
    new[3] = 20
    lens = [max(s + n + int(rng.integers(0, 200)), 1) for s, n in zip(lead, new)]
    b = Batch(rng, groups, lens, new, 2, 128, 64, typ, before=before, pad=1, layers=2, layer=1, crowd=crowd)
    b.check(b.attend(8, window, max_shared=hint, max_q=20 if hint else 0), window)


@pytest.mark.parametrize("typ,hd", [("f16", 128), ("q8", 64), ("f16", 64), ("q8", 128)])
def test_new_tokens_inside_the_shared_keys(typ, hd):
    """Sequences whose new tokens lie among the shared positions see no further than themselves; some end there, one
    has more new tokens than keys."""
    rng = np.random.default_rng(8)
    shared = 320
    new = [60, 1, 5, 300, 33, 20]
    lens = [330, 320, 100, 320, 321, 9]
    b = Batch(rng, [(6, shared)], lens, new, 2, hd, 32, typ, crowd=True)
    out = b.attend(4)
    at = np.concatenate([[0], np.cumsum(new)])
    assert not out[at[5]:at[5] + 11].any()  # before position 0
    out9 = out[at[5] + 11:at[6]]
    b.new, keep = b.new[:5], b.q
    b.check(out[: at[5]])
    keep = keep[: at[6]]
    ref, tol = attention(keep[at[5] + 11:], stored(b.k[5], typ), stored(b.v[5], typ), 9, np.float32(1 / math.sqrt(hd)))
    assert (np.abs(out9 - ref) <= tol).all()


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv_heads,hd,new,groups", [
    (8, 2, 128, 90, [(4, 700)]), (8, 2, 64, 90, [(4, 700), (2, 33), (5, 1500)]), (4, 4, 128, 300, [(5, 256)]),
    (16, 4, 128, 1, [(100, 1000)]), (8, 1, 64, 2, [(70, 900), (75, 64)]), (8, 2, 64, 40, [(40, 4500)])])
@pytest.mark.parametrize("window", [0, 300])
def test_many_rows(typ, heads, kv_heads, hd, new, groups, window):
    """Groups of many rows, over more than 64 sequences, and of many keys: ranges of several steps and of more than 64
    blocks."""
    rng = np.random.default_rng(new + hd)
    lead = [s for m, s in groups for _ in range(m)]
    n = [int(x) for x in rng.integers(1, new + 1, len(lead))]
    lens = [s + k + int(rng.integers(0, 100)) for s, k in zip(lead, n)]
    b = Batch(rng, groups, lens, n, kv_heads, hd, 32, typ, pad=3, crowd=True)
    b.check(b.attend(heads, window, grouped=False), window)  # at times as many partial rows either way
    b = Batch(rng, groups, lens, n, kv_heads, hd, 32, typ, pad=3)
    b.check(b.attend(heads, window, max_q=new, max_shared=max(lead)), window)


@pytest.mark.parametrize("typ,hd", [("f16", 64), ("q8", 128)])
@pytest.mark.parametrize("window", [2500, 4000, 4700])
def test_windows_inside_the_shared_keys(typ, hd, window):
    """Windows that begin among the shared keys, before a range or within it, and among the own ones."""
    rng = np.random.default_rng(window)
    lens = [4800 + int(x) for x in rng.integers(1, 90, 20)] + [2000 + int(x) for x in rng.integers(1, 700, 20)] + [4400]
    b = Batch(rng, [(20, 4800), (20, 2000)], lens, [1] * 40 + [3], 8, hd, 32, typ, crowd=True)
    b.check(b.attend(8, window, grouped=True), window)


@pytest.mark.parametrize("crowd", [False, True])
def test_many_groups(crowd):
    """More than 64 groups."""
    rng = np.random.default_rng(1)
    groups = [(int(rng.integers(0, 4)), int(rng.integers(0, 100))) for _ in range(150)]
    lead = [s for m, s in groups for _ in range(m)] + [0, 0]
    n = [int(x) for x in rng.integers(0, 3, len(lead))]
    lens = [max(1, s + k + int(rng.integers(0, 50))) for s, k in zip(lead, n)]
    b = Batch(rng, groups, lens, n, 1, 64, 32, "q8", crowd=crowd)
    b.check(b.attend(4))
    b.check(b.attend(4, max_shared=100))


def test_no_groups_and_in_place():
    rng = np.random.default_rng(2)
    b = Batch(rng, [], [70, 5, 200], [2, 1, 4], 2, 64, 32, "f16")
    b.check(b.attend(4))
    b = Batch(rng, [(3, 150)], [151, 170, 300], [1, 2, 40], 2, 64, 32, "f16", crowd=True)
    b.check(b.attend(4, in_place=True), padding=False)


def test_pages_and_rows_that_are_not_there():
    """A shared page outside the pool holds no keys; a NaN among the shared keys reaches who attends it alone."""
    rng = np.random.default_rng(3)
    new, lens, shared = [1, 2, 30], [200, 240, 190], 192
    b = Batch(rng, [(3, shared)], lens, new, 1, 64, 32, "f16", crowd=True)
    b.table[:3, 2] = [9999, -1, 1 << 30]
    present = [np.ones(n, bool) for n in b.lens]
    for p in present[:3]:
        p[64:96] = False
    b.check(b.attend(4), present=present)
    b = Batch(rng, [(3, shared)], lens, new, 1, 64, 32, "q8", crowd=True)
    for k in b.k[:3]:
        k[170, 0, 5] = np.nan  # the third sequence's first tokens stand before it
    b.fill()
    out = b.attend(4)
    assert np.isnan(out).any() and not np.isnan(out).all()
    b.check(out)


def test_large_scores_in_one_part():
    """Weights that all lie among the shared or all among the own keys."""
    rng = np.random.default_rng(4)
    for own in (0, 1):
        b = Batch(rng, [(3, 64)], [90, 100, 200], [1, 1, 3], 1, 64, 32, "f16", crowd=True)
        for k in b.k[:3]:
            (k[64:] if own else k[:64])[:] *= 30
        for i in (1, 2):
            b.k[i][:64] = b.k[0][:64]
        b.fill()
        b.check(b.attend(2))


def test_captured():
    """Replays take new lengths, groups and tables; without scratch every sequence reads its keys itself."""
    rng = np.random.default_rng(6)
    heads, page = 8, 32
    b = Batch(rng, [(3, 300), (2, 100)], [310, 340, 301, 180, 103, 40], [2, 1, 1, 3, 2, 1], 2, 64, page, "q8",
              crowd=True)
    b.arrays(heads)
    st = b.structs()
    nb = b.kv.attention_shared_scratch(*st, heads)
    assert nb > 0
    sc = torch.full((nb // 4 + 4,), float("nan"), device="cuda")
    other = torch.full_like(b.out, 7.0)
    q = b.d[5]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h = torch.cuda.current_stream().cuda_stream
        b.kv.attention_shared_dev(0, *st, q.data_ptr(), b.out.data_ptr(), heads, 1.0 / math.sqrt(64),
                                  scratch_ptr=sc.data_ptr(), scratch_bytes=nb, stream=h)
        b.kv.attention_shared_dev(0, *st, q.data_ptr(), other.data_ptr(), heads, 1.0 / math.sqrt(64), stream=h)
    for step in range(3):
        if step == 1:  # one key less each, the groups' borders moved
            b.lens = [n - 1 for n in b.lens]
            b.k, b.v = [x[:-1] for x in b.k], [x[:-1] for x in b.v]
            b.d[1].copy_(dev(b.lens, np.int32))
            b.d[4].copy_(dev([200, 64, 63], np.int32))
        if step == 2:
            b.d[3].copy_(dev([0, 3, 3, 5], np.int32))
            b.d[4].copy_(dev([200, 64, 60], np.int32))
        x = rng.standard_normal(b.q.shape).astype(np.float32)
        b.q = x
        q.copy_(dev(x))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.isnan(sc[nb // 4:]).all()
        b.check(b.out.cpu().numpy())
        b.check(other.cpu().numpy())
        b.check(b.again(heads, 0, 0))  # the program's own call in between


def test_stream_and_repeats():
    rng = np.random.default_rng(7)
    b = Batch(rng, [(9, 700)], [710 + 11 * i for i in range(9)], [1] * 9, 2, 128, 64, "f16", crowd=True)
    first = b.attend(8)
    b.check(first)
    s = torch.cuda.Stream()
    q = b.d[5]
    for _ in range(3):
        out = torch.zeros_like(b.out)
        torch.cuda.synchronize()
        b.kv.attention_shared_dev(0, *b.structs(), q.data_ptr(), out.data_ptr(), 8, 1 / math.sqrt(128),
                                  stream=s.cuda_stream)
        s.synchronize()
        assert np.array_equal(out.cpu().numpy(), first)


def test_refusals():
    b = Batch(np.random.default_rng(1), [(2, 40)], [50, 60], [1, 1], 2, 64, 32, "f16", crowd=True)
    b.arrays(4)
    bt, gr = b.structs()
    q, p = b.d[5].data_ptr(), b.d[0].data_ptr()

    def call(batch=bt, groups=gr, layer=0, qp=q, heads=4, scale=0.125, **kw):
        b.kv.attention_shared_dev(layer, batch, groups, qp, b.out.data_ptr(), heads, scale, **kw)

    sc = torch.zeros(64, device="cuda")
    for code, text, fn in ((-2, "-1 groups", lambda: call(groups=KVGroups(-1, p, p))),
                           (-2, "max_shared -1", lambda: call(groups=KVGroups(1, p, p, -1))),
                           (-1, "nil cu_seq", lambda: call(groups=KVGroups(1, 0, p))),
                           (-1, "nil cu_seq", lambda: call(groups=KVGroups(1, p, 0))),
                           (-1, "layer 1", lambda: call(layer=1)), (-1, "nil q", lambda: call(qp=0)),
                           (-2, "5 heads", lambda: call(heads=5)), (-1, "scale", lambda: call(scale=0.0)),
                           (-2, "under the row", lambda: call(q_stride=255)),
                           (-1, "16-byte", lambda: call(scratch_ptr=sc.data_ptr() + 4, scratch_bytes=1 << 20)),
                           (-2, "of scratch, needs", lambda: call(scratch_ptr=sc.data_ptr(), scratch_bytes=16)),
                           (-2, "-1 groups", lambda: b.kv.attention_shared_scratch(bt, KVGroups(-1, p, p), 4))):
        with pytest.raises(wv.WelvetError) as e:
            fn()
        assert e.value.code == code and text in str(e.value), str(e.value)
        assert "wv_kv_attention_shared" in str(e.value)
    wv.sync()
    assert (b.out == 7.0).all()
