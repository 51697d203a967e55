"""Pages of the paged KV cache on the device: sequences forked, resized and
emptied, pages copied and compacted, slots and positions of a batch, against a
table kept on the host one sequence after the other, and the cached rows
against what was written."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from welvet_amd.kv import KVBatch, KVCache, KVTables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def ints(x, t=np.int32):
    d = torch.from_numpy(np.ascontiguousarray(np.asarray(x, t))).cuda()
    torch.cuda.synchronize()
    return d


class Model:
    """The table as its definition says, sequence by sequence."""

    def __init__(self, seqs, width, pool, page):
        self.t = np.full((seqs, width), -1, np.int32)
        self.n, self.refs = np.zeros(seqs, np.int32), np.zeros(pool, np.int32)
        self.page, self.width = page, width
        self.ids = [[] for _ in range(seqs)]  # the rows that each sequence has written

    def held(self, n):
        return -(-int(n) // self.page)

    def fork(self, parent):
        t, n, ids = self.t.copy(), self.n.copy(), [list(x) for x in self.ids]
        for b, p in enumerate(parent):
            if p < -1 or p >= len(parent):
                continue
            self.t[b] = t[p] if p >= 0 else -1
            self.n[b] = n[p] if p >= 0 else 0
            self.ids[b] = list(ids[p]) if p >= 0 else []
        self.count()

    def count(self):
        self.refs[:] = 0
        for b, n in enumerate(self.n):
            np.add.at(self.refs, self.t[b, : self.held(n)], 1)

    def resize(self, to):
        ok = np.ones(len(to), np.int32)
        for b, m in enumerate(to):
            m = max(int(m), 0)
            if m < self.n[b]:
                for e in range(self.held(m), self.held(self.n[b])):
                    self.refs[self.t[b, e]] -= 1
                    self.t[b, e] = -1
                self.n[b] = m
                self.ids[b] = self.ids[b][:m]
        free = list(np.nonzero(self.refs == 0)[0])
        full = False
        for b, m in enumerate(to):
            m = max(int(m), 0)
            if m <= self.n[b]:
                continue
            if m > self.width * self.page:
                ok[b] = 0
                continue
            have, want = self.held(self.n[b]), self.held(m)
            last = self.t[b, have - 1] if self.n[b] % self.page else -1
            copy = int(last >= 0 and self.refs[last] > 1)
            full = full or want - have + copy > len(free)
            if full:
                ok[b] = 0
                continue
            if copy:
                self.refs[last] -= 1
            for e in range(have - copy, want):
                self.t[b, e] = free.pop(0)
                self.refs[self.t[b, e]] = 1
            self.n[b] = m
        return ok

    def compact(self):
        u = int((self.refs > 0).sum())
        holes = [p for p in range(u) if self.refs[p] == 0]
        moves = [p for p in range(u, len(self.refs)) if self.refs[p] > 0]
        for p, h in zip(moves, holes):
            self.t[self.t == p] = h
            self.refs[h], self.refs[p] = self.refs[p], 0
        return u


class Table:
    """A cache, a table on the device, and the model of both."""

    def __init__(self, seqs, width, pool, page, layers=2, kv_heads=2, hd=64, typ="f16"):
        self.kv = KVCache(layers, kv_heads, hd, page, pool, typ)
        self.m = Model(seqs, width, pool, page)
        self.layers, self.kv_heads, self.hd = layers, kv_heads, hd
        self.t, self.n, self.refs = ints(self.m.t), ints(self.m.n), ints(self.m.refs)
        self.work = torch.full((self.kv.tables_work(seqs, width),), 0x5a, dtype=torch.uint8, device="cuda")
        self.tables = KVTables(seqs, width, self.t.data_ptr(), self.n.data_ptr(), self.refs.data_ptr(),
                               self.work.data_ptr())
        self.next = 1

    def rows(self, ids, layer):
        """K and V of the written rows: whole numbers that fp16 codes hold exactly."""
        h, d = np.arange(self.kv_heads)[:, None], np.arange(self.hd)
        x = np.asarray(ids, np.int64)[:, None, None]
        k = (x * 7 + h * 31 + d * 3 + layer * 11) % 1021 + 1
        return k.astype(np.float32), ((k * 5 + 3) % 1019 + 1).astype(np.float32)

    def same(self):
        wv.sync()
        assert np.array_equal(self.n.cpu().numpy(), self.m.n), "lengths"
        assert np.array_equal(self.t.cpu().numpy(), self.m.t), "pages"
        assert np.array_equal(self.refs.cpu().numpy(), self.m.refs), "holders"

    def fork(self, parent):
        p = ints(parent)
        self.kv.fork_dev(self.tables, p.data_ptr())
        self.m.fork(parent)
        self.same()

    def resize(self, to):
        d, ok = ints(to), ints(np.full(len(to), 9))
        self.kv.resize_dev(self.tables, d.data_ptr(), ok.data_ptr())
        want = self.m.resize(to)
        self.same()
        assert np.array_equal(ok.cpu().numpy(), want)
        return want

    def compact(self):
        u = ints([-1])
        self.kv.compact_dev(self.tables, u.data_ptr())
        want = self.m.compact()
        self.same()
        assert int(u.cpu()[0]) == want

    def batch(self, new):
        cu = np.concatenate([[0], np.cumsum(new)])
        self.cu = ints(cu)
        return KVBatch(len(new), int(cu[-1]), self.m.width, self.cu.data_ptr(), self.n.data_ptr(), self.t.data_ptr())

    def slots(self, new):
        n = int(np.sum(new))
        s, p = ints(np.full(n, -7), np.int64), ints(np.full(n, -7))
        self.kv.slots_dev(self.batch(new), s.data_ptr(), p.data_ptr())
        wv.sync()
        want = np.concatenate([np.arange(self.m.n[b] - k, self.m.n[b]) for b, k in enumerate(new)]) if n else np.zeros(0)
        assert np.array_equal(p.cpu().numpy(), want)
        return s

    def write(self):
        """Rows of its own for whatever a sequence has grown by."""
        new = [int(n) - len(i) for n, i in zip(self.m.n, self.m.ids)]
        s = self.slots(new)
        for b, k in enumerate(new):
            self.m.ids[b] += list(range(self.next, self.next + k))
            self.next += k
        if not sum(new):
            return
        ids = np.concatenate([np.array(i[len(i) - k:], np.int64) for i, k in zip(self.m.ids, new)])
        for layer in range(self.layers):
            k, v = (torch.from_numpy(x).cuda() for x in self.rows(ids, layer))
            torch.cuda.synchronize()
            self.kv.write_dev(layer, k.data_ptr(), v.data_ptr(), s.data_ptr(), len(ids))
            wv.sync()

    def read(self):
        """Every sequence holds its rows, in every layer."""
        s = self.slots([int(n) for n in self.m.n])
        ids = np.concatenate([np.array(i, np.int64) for i in self.m.ids])
        if not ids.size:
            return
        for layer in range(self.layers):
            k, v = (torch.zeros(len(ids), self.kv_heads, self.hd, device="cuda") for _ in range(2))
            torch.cuda.synchronize()
            self.kv.read_dev(layer, s.data_ptr(), len(ids), k.data_ptr(), v.data_ptr())
            wv.sync()
            for got, want in zip((k, v), self.rows(ids, layer)):
                assert np.array_equal(got.cpu().numpy(), want), f"layer {layer}"


@pytest.mark.parametrize("typ,hd,kv_heads,page,layers", [("f16", 64, 2, 32, 2), ("f16", 128, 1, 128, 1),
                                                         ("f16", 128, 3, 64, 3)])
def test_fork_grow_write(typ, hd, kv_heads, page, layers):
    """Samples of one prompt, each with rows of its own behind it: a shared last page is copied before it is written."""
    for first in (1, page - 1, page, page + 1, 2 * page + 31, 2 * page + 32, 2 * page + 33):
        t = Table(5, 6, 40, page, layers, kv_heads, hd, typ)
        t.resize([first, 0, 3, 0, 0])
        t.write()
        t.fork([0, 0, 2, 0, -1])
        t.resize([first + 1, first + 2, 3, first, 0])  # 3 holds the last page on: both others copy it
        t.write()
        t.read()
        t.resize([first + 1, first + 3, 4, first + page, 0])
        t.write()
        t.read()
        t.fork([1, 2, 3, 0, 0])  # places traded
        t.resize([n + 1 for n in t.m.n])
        t.write()
        t.read()


@pytest.mark.parametrize("seqs,width", [(1, 1), (1, 130), (3, 65), (8, 33), (9, 700), (33, 40), (64, 31), (257, 9),
                                        (1025, 5), (4097, 3), (16384, 2)])
def test_fork_sizes(seqs, width):
    """Tables of all shapes: every row comes from where it should, and every page's holders are counted."""
    rng = np.random.default_rng(seqs)
    kv, pool = KVCache(1, 1, 64, 32, 2000, "f16"), 2000
    held = rng.integers(0, width + 1, seqs)
    t = np.where(np.arange(width) < held[:, None], rng.integers(0, pool, (seqs, width)), -1).astype(np.int32)
    refs = np.bincount(t[t >= 0], minlength=pool).astype(np.int32)
    dt, dn, dr = ints(t), ints(held * 32), ints(refs)
    tables = KVTables(seqs, width, dt.data_ptr(), dn.data_ptr(), dr.data_ptr(), dt.data_ptr())
    for _ in range(2):
        parent = rng.integers(-2, seqs + 1, seqs).astype(np.int32)  # some are emptied, some outside the table
        d = ints(parent)
        kv.fork_dev(tables, d.data_ptr())
        wv.sync()
        stay = (parent < -1) | (parent >= seqs)
        src = np.where(stay, np.arange(seqs), np.maximum(parent, 0))
        t, held = np.where((parent == -1)[:, None], -1, t[src]), np.where(parent == -1, 0, held[src])
        assert np.array_equal(dt.cpu().numpy(), t) and np.array_equal(dn.cpu().numpy(), held * 32)
        assert np.array_equal(dr.cpu().numpy(), np.bincount(t[t >= 0], minlength=pool))


@pytest.mark.parametrize("seqs,width,pool,page,seed", [(1, 4, 3, 32, 0), (7, 9, 41, 32, 1), (70, 5, 200, 64, 2),
                                                       (1500, 3, 2300, 32, 3), (33, 40, 9000, 32, 4)])
def test_random_calls(seqs, width, pool, page, seed):
    """Forks, sizes, ends and compactions in any order, with pools that run out."""
    rng = np.random.default_rng(seed)
    t = Table(seqs, width, pool, page, layers=1, kv_heads=1)
    for step in range(8):
        kind = step % 4
        if kind in (0, 2):
            top = width * page + (1 if step == 2 else 0)  # at times more than the table has room for
            to = np.where(rng.random(seqs) < 0.4, t.m.n, rng.integers(-1, top + 1, seqs))
            t.resize(to)
            t.write()
        elif kind == 1:
            parent = np.where(rng.random(seqs) < 0.5, np.arange(seqs), rng.integers(-2, seqs + 1, seqs))
            t.fork(parent)
        else:
            t.compact()
        t.read()


def test_pool_runs_out_in_order():
    """The first that does not fit stops the growing ones behind it, even ones that need no page; shrinking ones go on."""
    t = Table(5, 8, 6, 32)
    t.resize([64, 10, 0, 70, 0])
    t.write()
    ok = t.resize([65, 10, 33, 20, 5])
    assert ok.tolist() == [1, 1, 0, 1, 0]
    assert t.resize([66, 11, 200, 21, 0]).tolist() == [1, 1, 0, 0, 1]
    t.write()
    t.read()


def test_all_holders_grow():
    """Of sequences that are all holders of a last page and all grow, the last one keeps it."""
    t = Table(3, 3, 9, 32)
    t.resize([40, 0, 0])
    t.write()
    t.fork([0, 0, 0])
    last = int(t.m.t[0, 1])
    t.resize([41, 41, 41])
    assert t.m.t[2, 1] == last and t.m.refs[last] == 1
    t.write()
    t.read()


def test_pages_outside_the_pool():
    """Entries that name no page of the pool are carried along and count for nothing; their rows have no slot."""
    t = Table(3, 4, 8, 32)
    t.resize([100, 40, 0])
    t.m.t[0, 1] = 99
    t.m.t[1, 1] = -5
    t.m.refs[1] = 0
    t.m.refs[5] = 0
    t.t.copy_(ints(t.m.t))
    t.refs.copy_(ints(t.m.refs))
    torch.cuda.synchronize()
    p = ints([0, 1, 0])
    t.kv.fork_dev(t.tables, p.data_ptr())
    wv.sync()
    assert t.t.cpu().numpy()[2].tolist() == [0, 99, 2, 3]
    assert t.refs.cpu().numpy().tolist() == [2, 0, 2, 2, 1, 0, 0, 0]
    d, ok = ints([100, 41, 10]), ints([0, 0, 0])
    t.kv.resize_dev(t.tables, d.data_ptr(), ok.data_ptr())
    u = ints([0])
    t.kv.compact_dev(t.tables, u.data_ptr())
    wv.sync()
    assert t.t.cpu().numpy()[:, :2].tolist() == [[0, 99], [1, -5], [0, -1]] and int(u.cpu()[0]) == 4
    t.m.n[:] = [100, 41, 10]
    s = t.slots([100, 41, 10]).cpu().numpy()
    assert (s[32:64] == -1).all() and (s[132:141] == -1).all() and (s[:32] == np.arange(32)).all()


def test_slots_edges():
    """Padding rows, empty sequences, more new tokens than positions, positions past the table."""
    t = Table(4, 2, 8, 32)
    t.resize([64, 33, 0, 5])
    ln, cu = ints([70, 33, 0, 2]), ints([0, 8, 8, 9, 13])
    b = KVBatch(4, 15, 2, cu.data_ptr(), ln.data_ptr(), t.t.data_ptr())
    s, p = ints(np.full(15, 5), np.int64), ints(np.full(15, 5))
    t.kv.slots_dev(b, s.data_ptr(), p.data_ptr())
    wv.sync()
    base = t.m.t.astype(np.int64) * 32
    assert p.cpu().numpy().tolist() == list(range(62, 70)) + [-1] + [-2, -1, 0, 1] + [0, 0]
    want = [base[0, 1] + 30, base[0, 1] + 31] + [-1] * 6 + [-1] + [-1, -1, base[3, 0], base[3, 0] + 1] + [-1, -1]
    assert s.cpu().numpy().tolist() == want
    t.kv.slots_dev(b, s.data_ptr())  # without positions
    wv.sync()
    assert s.cpu().numpy().tolist() == want


@pytest.mark.parametrize("seqs", [4096, 4097, 20000])
def test_slots_of_many_sequences(seqs):
    rng = np.random.default_rng(seqs)
    kv = KVCache(1, 1, 64, 32, 50)
    new = rng.integers(0, 3, seqs)
    ln = new + rng.integers(0, 60, seqs)
    table = rng.integers(-1, 51, (seqs, 2)).astype(np.int32)
    cu, dl, dt = ints(np.concatenate([[0], np.cumsum(new)])), ints(ln), ints(table)
    n = int(new.sum()) + 3
    s, p = ints(np.zeros(n), np.int64), ints(np.zeros(n))
    kv.slots_dev(KVBatch(seqs, n, 2, cu.data_ptr(), dl.data_ptr(), dt.data_ptr()), s.data_ptr(), p.data_ptr())
    wv.sync()
    b = np.repeat(np.arange(seqs), new)
    q = ln[b] - new[b] + np.concatenate([np.arange(k) for k in new])
    page = table[b, np.minimum(q // 32, 1)].astype(np.int64)
    want = np.where((page >= 0) & (page < 50), page * 32 + q % 32, -1)
    assert np.array_equal(p.cpu().numpy(), np.concatenate([q, [0, 0, 0]]))
    assert np.array_equal(s.cpu().numpy(), np.concatenate([want, [-1, -1, -1]]))


@pytest.mark.parametrize("typ", ["f16", "q8"])
def test_copy_pages(typ):
    kv = KVCache(3, 2, 128, 64, 9, typ)
    rng = np.random.default_rng(5)
    x = [[torch.from_numpy(rng.standard_normal((9 * 64, 2, 128)).astype(np.float32)).cuda() for _ in range(2)]
         for _ in range(3)]
    slots = ints(np.arange(9 * 64), np.int64)
    for layer in range(3):
        kv.write_dev(layer, x[layer][0].data_ptr(), x[layer][1].data_ptr(), slots.data_ptr(), 9 * 64)

    def read(layer):
        k, v = (torch.zeros(9 * 64, 2, 128, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        kv.read_dev(layer, slots.data_ptr(), 9 * 64, k.data_ptr(), v.data_ptr())
        wv.sync()
        return k.view(9, 64, 2, 128), v.view(9, 64, 2, 128)

    before = [read(i) for i in range(3)]
    src, dst = ints([0, 8, 0, -1, 3, 9, 5]), ints([4, 1, 7, 2, 40, 2, 5])
    kv.copy_pages_dev(src.data_ptr(), dst.data_ptr(), 7)
    order = [0, 8, 2, 3, 0, 5, 6, 0, 8]
    for i in range(3):
        for a, b in zip(before[i], read(i)):
            assert torch.equal(a[order], b)


def test_captured_step():
    """A step of a graph: forked, grown, slots taken, replayed with the program's own calls in between."""
    page = 32
    t = Table(4, 8, 40, page)
    t.resize([35, 0, 0, 0])
    t.write()
    parent, to, ok = ints([0, 0, 0, 3]), ints([36, 36, 36, 2]), ints([0, 0, 0, 0])
    slots, pos = ints(np.zeros(4), np.int64), ints(np.zeros(4))
    b, cu = t.batch([1, 1, 1, 1]), t.cu  # cu stays: the graph reads it
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        h = torch.cuda.current_stream().cuda_stream
        t.kv.fork_dev(t.tables, parent.data_ptr(), stream=h)
        t.kv.resize_dev(t.tables, to.data_ptr(), ok.data_ptr(), stream=h)
        t.kv.slots_dev(b, slots.data_ptr(), pos.data_ptr(), stream=h)
    for step in range(3):
        want = [36 + step] * 3 + [2 + step]
        to.copy_(ints(want))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t.m.fork([0, 0, 0, 3])
        assert t.m.resize(want).all()
        t.same()
        assert pos.cpu().numpy().tolist() == [n - 1 for n in want]
        got = slots.cpu().numpy()
        assert got.tolist() == [int(t.m.t[i, (n - 1) // page]) * page + (n - 1) % page for i, n in enumerate(want)]
        t.write()
        t.compact()
        t.read()
    del g, cu


def test_refusals():
    kv = KVCache(1, 1, 64, 32, 4)
    z = ints(np.zeros(64))
    p = z.data_ptr()
    with pytest.raises(wv.WelvetError) as e:
        kv.tables_work(16385, 1)
    assert e.value.code == -2 and "at most 16384" in str(e.value)
    with pytest.raises(wv.WelvetError) as e:
        kv.tables_work(1, 1 << 26)
    assert e.value.code == -2 and "2^31" in str(e.value)
    good = KVTables(1, 1, p, p, p, p)
    for bad in (KVTables(1, 1, 0, p, p, p), KVTables(1, 1, p, 0, p, p), KVTables(1, 1, p, p, 0, p),
                KVTables(1, 1, p, p, p, 0)):
        for call in (lambda t: kv.fork_dev(t, p), lambda t: kv.resize_dev(t, p, p), lambda t: kv.compact_dev(t)):
            with pytest.raises(wv.WelvetError) as e:
                call(bad)
            assert e.value.code == -1 and "nil pages" in str(e.value)
    for call, word in ((lambda: kv.fork_dev(good, 0), "nil parent"), (lambda: kv.resize_dev(good, 0, p), "nil len"),
                       (lambda: kv.resize_dev(good, p, 0), "nil len"), (lambda: kv.copy_pages_dev(0, p, 1), "nil src"),
                       (lambda: kv.slots_dev(KVBatch(1, 1, 1, p, p, p), 0), "nil slots"),
                       (lambda: kv.slots_dev(KVBatch(1, 1, 1, p, p, 0), p), "nil slots")):
        with pytest.raises(wv.WelvetError) as e:
            call()
        assert e.value.code == -1 and word in str(e.value)
    with pytest.raises(wv.WelvetError) as e:
        kv.copy_pages_dev(p, p, -1)
    assert e.value.code == -2
    with pytest.raises(wv.WelvetError) as e:
        kv.slots_dev(KVBatch(1, -1, 1, p, p, p), p)
    assert e.value.code == -2
    none = KVTables(0, 0, 0, 0, 0, 0)  # nothing to do
    kv.fork_dev(none, 0)
    kv.resize_dev(none, 0, 0)
    kv.compact_dev(none)
    kv.copy_pages_dev(0, 0, 0)
    kv.slots_dev(KVBatch(0, 0, 0, 0, 0, 0), 0)
