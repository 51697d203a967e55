"""A serving step of a batch as its calls are used together: the table grown (with forks, ends and a compaction between
steps), slots and positions, Q, K and V projections with every request's adapters, rotary positions, the rows written,
attention that reads shared prefixes once, and the output projection with its adapters. All of a step goes to one
stream, or is replayed from a graph; afterwards each call's results are checked in float64 on what it was given."""
import math
import threading

import numpy as np
import pytest
import torch

import welvet_amd as wv
from kv_ref import attention, stored
from test_gpu_adapters import U, held
from test_gpu_kv_pages import Model
from test_gpu_rope import check as check_rope, freqs
from welvet_amd.adapters import AdapterBatch, Adapters, apply_dev, scratch
from welvet_amd.kv import KVBatch, KVCache, KVGroups, KVTables
from welvet_amd.rope import Rope

pytestmark = pytest.mark.gpu
HID, HEADS, KV, HD, PAGE = 256, 8, 2, 64, 32
SEQS, WIDTH, POOL, MOST = 70, 2048, 900, 200  # rows of a table, pages of one, pages of the pool, token rows of a step


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


class Step:
    def __init__(self, typ, seed):
        rng = self.rng = np.random.default_rng(seed)
        self.typ = typ
        dims = [HEADS * HD, KV * HD, KV * HD, HID]
        self.blobs = [wv.upload(wv.pack("Q8_0", (rng.standard_normal(o * i) / np.sqrt(i)).astype(np.float32), o, i))
                      for o, i in zip(dims, (HID, HID, HID, HEADS * HD))]
        self.sets, self.w = [], []
        for o, i in zip(dims, (HID, HID, HID, HEADS * HD)):
            s, w = Adapters(o, i, 16, 3), []
            for j, r in enumerate((16, 5, 8)):
                a, av = held(rng.standard_normal((r, i)) / np.sqrt(i), "bf16")
                b, bv = held(rng.standard_normal((o, r)) * 0.3, "bf16")
                s.set(j, a, b, 0.5 + j)
                w.append((av, bv, 0.5 + j))
            self.sets.append(s)
            self.w.append(w)
        self.rope = Rope(HD, theta=1e4, scaling="ramp_turns", factor=4.0, trained=64, low=1.0, high=4.0)
        self.f = freqs(HD, 1e4, "ramp_turns", 4.0, 64, 1.0, 4.0)
        self.kv = KVCache(1, KV, HD, PAGE, POOL, typ)
        self.m = Model(SEQS, WIDTH, POOL, PAGE)
        self.rows = [[np.zeros((0, KV, HD), np.float32)] * 2 for _ in range(SEQS)]  # K and V as written
        self.table = torch.full((SEQS, WIDTH), -1, dtype=torch.int32, device="cuda")
        i32 = dict(dtype=torch.int32)
        self.len, self.refs, self.to, self.ok = zeros(SEQS, **i32), zeros(POOL, **i32), zeros(SEQS, **i32), zeros(SEQS, **i32)
        self.parent, self.cu, self.which = zeros(SEQS, **i32), zeros(SEQS + 1, **i32), zeros(SEQS, **i32)
        self.group_cu, self.shared = zeros(4, **i32), zeros(3, **i32)
        self.work = torch.empty(self.kv.tables_work(SEQS, WIDTH), dtype=torch.uint8, device="cuda")
        self.tables = KVTables(SEQS, WIDTH, self.table.data_ptr(), self.len.data_ptr(), self.refs.data_ptr(),
                               self.work.data_ptr())
        self.x = zeros(MOST, HID)
        self.base = [zeros(MOST, o) for o in dims]
        self.y = [zeros(MOST, o) for o in dims]
        self.q, self.k = zeros(MOST, HEADS, HD), zeros(MOST, KV, HD)
        self.att = zeros(MOST, HEADS, HD)
        self.slots, self.pos = zeros(MOST, dtype=torch.int64), zeros(MOST, **i32)
        self.batch = KVBatch(SEQS, MOST, WIDTH, self.cu.data_ptr(), self.len.data_ptr(), self.table.data_ptr())
        self.groups = KVGroups(3, self.group_cu.data_ptr(), self.shared.data_ptr())
        self.ab = AdapterBatch(SEQS, MOST, self.cu.data_ptr(), self.which.data_ptr())
        na = self.kv.attention_shared_scratch(self.batch, self.groups, HEADS)
        assert na != self.kv.attention_scratch(self.batch, HEADS)  # shared keys are read once
        self.sa = torch.empty(na, dtype=torch.uint8, device="cuda")
        self.sd = torch.empty(max(scratch(self.sets[:3], self.ab), scratch(self.sets[3:], self.ab)), dtype=torch.uint8,
                              device="cuda")
        torch.cuda.synchronize()

    def enqueue(self, h, mine=True):
        """mine: with scratch of the step's own, else the library's."""
        p = lambda t: t.data_ptr()  # noqa: E731
        own = dict(scratch_ptr=p(self.sd), scratch_bytes=self.sd.numel(), stream=h) if mine else dict(stream=h)
        att = dict(scratch_ptr=p(self.sa), scratch_bytes=self.sa.numel(), stream=h) if mine else dict(stream=h)
        self.kv.resize_dev(self.tables, p(self.to), p(self.ok), stream=h)
        self.kv.slots_dev(self.batch, p(self.slots), p(self.pos), stream=h)
        for i in range(3):
            self.blobs[i].matvec_dev(p(self.x), p(self.base[i]), MOST, stream=h)
        apply_dev(self.sets[:3], self.ab, p(self.x), [p(t) for t in self.y[:3]], base_ptrs=[p(t) for t in self.base[:3]],
                  **own)
        self.rope.apply_dev(p(self.pos), MOST, p(self.y[0]), HEADS, p(self.y[1]), KV, q_out_ptr=p(self.q),
                            k_out_ptr=p(self.k), stream=h)
        self.kv.write_dev(0, p(self.k), p(self.y[2]), p(self.slots), MOST, stream=h)
        self.kv.attention_shared_dev(0, self.batch, self.groups, p(self.q), p(self.att), HEADS, 1 / math.sqrt(HD),
                                     **att)
        self.blobs[3].matvec_dev(p(self.att), p(self.base[3]), MOST, stream=h)
        apply_dev(self.sets[3:], self.ab, p(self.att), [p(self.y[3])], base_ptrs=[p(self.base[3])], **own)

    def inputs(self, new, which, group_cu, shared):
        """New tokens and adapter of each sequence, the groups."""
        self.new, self.ids = new, which
        self.to.copy_(torch.tensor(self.m.n + np.array(new), dtype=torch.int32))
        self.cu.copy_(torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)))
        self.which.copy_(torch.tensor(which, dtype=torch.int32))
        self.group_cu.copy_(torch.tensor(group_cu, dtype=torch.int32))
        self.shared.copy_(torch.tensor(shared, dtype=torch.int32))
        self.x.copy_(torch.from_numpy(self.rng.standard_normal((MOST, HID)).astype(np.float32)))
        torch.cuda.synchronize()

    def check_adapters(self, i, x, at):
        """Rows of set i: base + scale B (A x)."""
        base, y = self.base[i].cpu().numpy(), self.y[i].cpu().numpy()
        for b, n in enumerate(self.new):
            rows, a = slice(at[b], at[b + 1]), self.ids[b]
            want, tol = base[rows].astype(np.float64), 0.0
            if 0 <= a < 3:
                A, B, s = self.w[i][a]
                xx = x[rows].astype(np.float64)
                h = xx @ A.T
                want = want + s * (h @ B.T)
                tol = s * ((x.shape[1] / 4 + 64) * U * (np.abs(xx) @ np.abs(A).T) @ np.abs(B).T
                           + 20 * U * np.abs(h) @ np.abs(B).T) + 2 * U * np.abs(want)
            assert (np.abs(y[rows] - want) <= tol).all(), f"set {i}, sequence {b}"

    def check(self):
        """After a step: every call's results on what it was given."""
        ok = self.m.resize(self.m.n + np.array(self.new))
        assert np.array_equal(self.ok.cpu().numpy(), ok) and ok.all()
        for got, want in ((self.table, self.m.t), (self.len, self.m.n), (self.refs, self.m.refs)):
            assert np.array_equal(got.cpu().numpy(), want)
        at = np.concatenate([[0], np.cumsum(self.new)])
        n = int(at[-1])
        pos = np.concatenate([np.arange(self.m.n[b] - k, self.m.n[b]) for b, k in enumerate(self.new)])
        assert np.array_equal(self.pos.cpu().numpy(), np.concatenate([pos, np.zeros(MOST - n)]))
        assert (self.slots.cpu().numpy()[n:] == -1).all()
        x = self.x.cpu().numpy()
        for i in range(3):
            self.check_adapters(i, x, at)
        y = [t.cpu().numpy()[:n] for t in self.y]
        q, k = self.q.cpu().numpy()[:n], self.k.cpu().numpy()[:n]
        check_rope(q, y[0].reshape(n, HEADS, HD), pos, self.f, "half", HD, 1.0)
        check_rope(k, y[1].reshape(n, KV, HD), pos, self.f, "half", HD, 1.0)
        v, att = y[2].reshape(n, KV, HD), self.att.cpu().numpy()
        for b, cnt in enumerate(self.new):
            rows = slice(at[b], at[b + 1])
            self.rows[b] = [np.concatenate([old, t[rows]]) for old, t in zip(self.rows[b], (k, v))]
            ref, tol = attention(q[rows], stored(self.rows[b][0], self.typ), stored(self.rows[b][1], self.typ), cnt,
                                 np.float32(1 / math.sqrt(HD)))
            assert (np.abs(att[rows] - ref) <= tol).all(), f"attention of sequence {b}"
        self.check_adapters(3, att.reshape(MOST, HEADS * HD), at)

    def fork(self, parent):
        self.parent.copy_(torch.tensor(parent, dtype=torch.int32))
        torch.cuda.synchronize()
        self.kv.fork_dev(self.tables, self.parent.data_ptr())
        wv.sync()
        self.m.fork(parent)
        old = [list(r) for r in self.rows]
        for b, p in enumerate(parent):
            self.rows[b] = old[p] if p >= 0 else [np.zeros((0, KV, HD), np.float32)] * 2

    def compact(self):
        self.kv.compact_dev(self.tables)
        wv.sync()
        self.m.compact()


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("graph", [False, True])
def test_steps(typ, graph):
    s = Step(typ, 3)
    stream, g = torch.cuda.Stream(), None
    which = [(b % 5) - 1 for b in range(SEQS)]  # none, 0, 1, 2, and one that no set knows

    def step(new, group_cu, shared):
        nonlocal g
        s.inputs(new, which, group_cu, shared)
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
        s.check()

    def of(**new):
        return [new.get(f"s{b}", 0) for b in range(SEQS)]

    # two prompts of their own
    step(of(s0=100, s40=77), [0, 0, 0, 0], [0, 0, 0])
    # 30 answers to the first, 20 to the second; the others stay idle
    s.fork([0 if b < 30 else 40 if 40 <= b < 60 else -1 for b in range(SEQS)])
    step([1] * 30 + [0] * 10 + [1] * 20 + [0] * 10, [0, 30, 40, 60], [100, 0, 77])
    # some trade places, two end, one new prompt starts beside the single tokens
    order = [b for b in range(SEQS)]
    order[3], order[5], order[7], order[41], order[59] = 5, 3, -1, 40, -1
    s.fork(order)
    s.compact()
    new = [2 if b % 3 == 0 else 1 for b in range(30)] + [0] * 10 + [1] * 20 + [50] + [0] * 9
    new[7] = new[59] = 0
    step(new, [0, 30, 40, 60], [100, 32, 77])
    # the same again, with the groups the other way round: fewer shared positions, one group more
    new = [1] * 30 + [0] * 10 + [3] * 20 + [1] + [0] * 9
    new[7] = new[59] = 0
    step(new, [0, 15, 30, 60], [99, 100, 0])


def test_threads():
    """Steps of several batches at once, each from a host thread and on a stream of its own, in the library's scratch."""
    steps = [Step("f16", seed) for seed in (5, 6, 7)]
    new = [1] * 40 + [0] * 10 + [2] * 20
    for s in steps:
        s.inputs([100] + [0] * 39 + [60] + [0] * 29, [0] * SEQS, [0] * 4, [0] * 3)
        s.enqueue(None)
        wv.sync()
        s.check()
        s.fork([0 if b < 40 else 40 for b in range(SEQS)])
        s.inputs(new, [(b % 4) - 1 for b in range(SEQS)], [0, 40, 70, 70], [100, 60, 0])
    failed = []

    def run(s):
        try:
            st = torch.cuda.Stream()
            for _ in range(20):  # the same call, so the same results; the lengths are there after the first
                s.enqueue(st.cuda_stream, False)
            st.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(s,)) for s in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for s in steps:
        s.check()
