"""Steps whose pool runs out, with the batch laid out for all sequences: a refused sequence's new rows are written
nowhere, so what it holds, and what others that share its pages hold and attend over, stays."""
import ctypes

import numpy as np
import pytest
import torch

import welvet_amd as wv
from kv_ref import attention, stored
from test_gpu_kv_pages import Table, ints
from welvet_amd.kv import KVBatch, KVGroups

pytestmark = pytest.mark.gpu
HEADS, LAYERS, PAGE = 4, 2, 32


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


class Step:
    """`seqs` sequences that each want new[b] more rows a step; the rows' numbers are known before who is served is."""

    def __init__(self, seqs, width, pool, new, pad=0):
        self.t = Table(seqs, width, pool, PAGE, layers=LAYERS)
        self.seqs, self.rows = seqs, sum(new) + pad
        self.cu, self.to, self.ok = ints(np.zeros(seqs + 1)), ints(np.zeros(seqs)), ints(np.zeros(seqs))
        self.slots, self.pos = ints(np.zeros(self.rows), np.int64), ints(np.zeros(self.rows))
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        t = self.t
        self.kv = [[f(self.rows, t.kv_heads, t.hd) for _ in range(2)] for _ in range(LAYERS)]
        self.q, self.out = f(self.rows, HEADS, t.hd), f(self.rows, HEADS, t.hd)
        self.gc, self.sh = ints([0, seqs]), ints([0])
        self.batch = KVBatch(seqs, self.rows, width, self.cu.data_ptr(), t.n.data_ptr(), t.t.data_ptr())
        self.groups = KVGroups(1, self.gc.data_ptr(), self.sh.data_ptr())
        self.scratch = torch.zeros(max(t.kv.attention_shared_scratch(self.batch, self.groups, HEADS), 16),
                                   dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def inputs(self, new, shared, seed):
        self.new, t = new, self.t
        self.want = t.m.n + np.array(new)
        self.ids, at = [], t.next
        for k in new:
            self.ids.append(list(range(at, at + k)))
            at += k
        t.next = at
        self.cu.copy_(ints(np.concatenate([[0], np.cumsum(new)])))
        self.to.copy_(ints(self.want))
        self.sh.copy_(ints([shared]))
        n = sum(new)
        for layer in range(LAYERS):
            for d, x in zip(self.kv[layer], t.rows(sum(self.ids, []), layer)):
                d[:n].copy_(torch.from_numpy(x))
        self.q.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal(self.q.shape).astype(np.float32)))
        torch.cuda.synchronize()

    def enqueue(self, h):
        t, p = self.t, lambda x: x.data_ptr()  # noqa: E731
        t.kv.resize_dev(t.tables, p(self.to), p(self.ok), stream=h)
        t.kv.slots_dev(self.batch, p(self.slots), p(self.pos), stream=h, ok_ptr=p(self.ok))
        for layer, (k, v) in enumerate(self.kv):
            t.kv.write_dev(layer, p(k), p(v), p(self.slots), self.rows, stream=h)
        t.kv.attention_shared_dev(LAYERS - 1, self.batch, self.groups, p(self.q), p(self.out), HEADS,
                                  1e-3, scratch_ptr=p(self.scratch), scratch_bytes=self.scratch.numel(), stream=h)

    def check(self):
        """Tables, slots, positions, all rows of all sequences, the attention of those that were served."""
        t = self.t
        ok = t.m.resize(self.want)
        t.same()
        assert np.array_equal(self.ok.cpu().numpy(), ok)
        slots, pos = self.slots.cpu().numpy(), self.pos.cpu().numpy()
        at = np.concatenate([[0], np.cumsum(self.new)])
        for b, k in enumerate(self.new):
            rows = slice(at[b], at[b + 1])
            if not ok[b]:
                assert (slots[rows] == -1).all() and (pos[rows] == 0).all(), f"refused sequence {b}"
                continue
            j = np.arange(t.m.n[b] - k, t.m.n[b])
            assert np.array_equal(pos[rows], j)
            assert np.array_equal(slots[rows], t.m.t[b, j // PAGE].astype(np.int64) * PAGE + j % PAGE)
            t.m.ids[b] += self.ids[b]
        assert (slots[at[-1]:] == -1).all() and (pos[at[-1]:] == 0).all()
        t.read()
        q, out = self.q.cpu().numpy(), self.out.cpu().numpy()
        for b, k in enumerate(self.new):
            if not ok[b]:
                continue
            rows = slice(at[b], at[b + 1])
            kk, vv = (stored(x, "f16") for x in t.rows(t.m.ids[b], LAYERS - 1))
            ref, tol = attention(q[rows], kk, vv, k, np.float32(1e-3))
            assert (np.abs(out[rows] - ref) <= tol).all(), f"attention of sequence {b}"
        return ok.tolist()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("length", [64, 40, 63, 65, 33])
@pytest.mark.parametrize("new", [[1] * 4, [3, 1, 0, 2], [40, 2, 33, 1]])
def test_forked_sequences(length, new, graph):
    """Four samples of one prompt whose last page is full or not, as many free pages as the first of them needs; then it
    ends, and of those that were refused some are served."""
    held = -(-length // PAGE)
    first = -(-(length + new[0]) // PAGE) - length // PAGE  # pages that the first one takes
    s = Step(4, 8, held + first, new, pad=2)
    t = s.t
    t.resize([length, 0, 0, 0])
    t.write()
    t.fork([0, 0, 0, 0])
    g, stream = None, torch.cuda.Stream()

    def step(new, seed, shared=length):
        nonlocal g
        s.inputs(new, shared, seed)
        if graph and g is None:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                s.enqueue(torch.cuda.current_stream().cuda_stream)
        if graph:
            g.replay()
            torch.cuda.synchronize()
        else:
            s.enqueue(stream.cuda_stream)
            stream.synchronize()
        return s.check()

    ok = step(new, 1)
    assert ok[0] == 1 and not all(ok)
    again = [0 if ok[b] else k for b, k in enumerate(new)]  # who waits asks again, in vain
    assert not all(step(again, 2))
    t.fork([-1, 1, 2, 3])
    step([0] + again[1:], 3, 0)


def test_more_rows_than_the_table_has_room_for():
    """Refused for the table's width: the others are served, that one's rows stay."""
    s = Step(2, 2, 9, [2, 2])
    s.t.resize([63, 5])
    s.t.write()
    s.inputs([2, 2], 0, 1)
    s.enqueue(None)
    wv.sync()
    assert s.check() == [0, 1]


def test_slots_without_refusals():
    """With every sequence served, the same as without being told; many sequences of which some were refused."""
    rng = np.random.default_rng(2)
    for seqs in (5, 4096, 4097, 9000):
        t = Table(1, 1, 50, PAGE, layers=1, kv_heads=1)
        new = rng.integers(0, 3, seqs)
        ln = new + rng.integers(0, 60, seqs)
        table, cu, dl = ints(rng.integers(-1, 51, (seqs, 2))), ints(np.concatenate([[0], np.cumsum(new)])), ints(ln)
        n = int(new.sum()) + 3
        b = KVBatch(seqs, n, 2, cu.data_ptr(), dl.data_ptr(), table.data_ptr())
        got = []
        refused = rng.random(seqs) < 0.3
        for ok in (None, np.ones(seqs), np.where(refused, 0, 7)):
            s, p = ints(np.full(n, -7), np.int64), ints(np.full(n, -7))
            d = None if ok is None else ints(ok)
            t.kv.slots_dev(b, s.data_ptr(), p.data_ptr(), ok_ptr=None if d is None else d.data_ptr())
            wv.sync()
            got.append((s.cpu().numpy(), p.cpu().numpy()))
        assert all(np.array_equal(x, y) for x, y in zip(got[0], got[1]))
        hit = np.concatenate([np.repeat(refused, new), [False] * 3])
        assert np.array_equal(got[2][0], np.where(hit, -1, got[0][0]))
        assert np.array_equal(got[2][1], np.where(hit, 0, got[0][1]))


def test_refusals():
    t = Table(1, 1, 4, PAGE)
    z = ints(np.zeros(4))
    L, p = wv.lib(), z.data_ptr()
    b = KVBatch(1, 1, 1, p, p, p)
    assert L.wv_kv_slots_served_dev(t.kv.handle, ctypes.byref(b), None, p, p, None) == -1
    assert b"wv_kv_slots_served: nil ok" in L.wv_last_error()
    assert L.wv_kv_slots_served_dev(t.kv.handle, None, p, p, p, None) == -1
    assert L.wv_kv_slots_served_dev(t.kv.handle, ctypes.byref(KVBatch(1, -1, 1, p, p, p)), p, p, p, None) == -2
    assert L.wv_kv_slots_served_dev(t.kv.handle, ctypes.byref(KVBatch(0, 0, 0, 0, 0, 0)), None, None, None, None) == 0
