"""Low-rank adapters on the device against float64."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from welvet_amd.adapters import AdapterBatch, Adapters, apply_dev, scratch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def dev(x):
    d = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    torch.cuda.synchronize()
    return d


def held(x, typ):
    """16-bit values of x, as bits and in f64."""
    t = torch.from_numpy(np.asarray(x, np.float32)).to(torch.float16 if typ == "f16" else torch.bfloat16)
    return t.view(torch.int16).numpy().view(np.uint16), t.double().numpy()


class Case:
    def __init__(self, rng, sets, cols, ranks, new, which, typ="bf16", max_rank=None, pad=0):
        """sets: output rows of each; ranks of the adapters; tokens and adapter of each sequence."""
        self.rng, self.cols, self.new, self.which, self.rows = rng, cols, new, which, sets
        self.t = sum(new) + pad
        self.sets, self.w = [], []
        for o in sets:
            s = Adapters(o, cols, max_rank or max(ranks), len(ranks), typ)
            w = []
            for j, r in enumerate(ranks):
                if r == 0:
                    w.append(None)
                    continue
                a, av = held(rng.standard_normal((r, cols)) / np.sqrt(cols), typ)
                b, bv = held(rng.standard_normal((o, r)) * 0.4, typ)
                scale = float(np.float32(rng.uniform(0.3, 2.0)))
                s.set(j, a, b, scale)
                w.append((av, bv, scale))
            self.sets.append(s)
            self.w.append(w)
        self.x = rng.standard_normal((self.t, cols)).astype(np.float32)
        self.base = [rng.standard_normal((self.t, o)).astype(np.float32) for o in sets]
        self.cu, self.ids = dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), dev(np.array(which, np.int32))
        self.batch = AdapterBatch(len(new), self.t, self.cu.data_ptr(), self.ids.data_ptr(), max(new, default=0))

    def want(self, i):
        """Rows of set i, and a bound on each value's error. h = A x sums products that are rounded once each, in
        chains of at most a quarter of the columns (or 16) that are then joined by 40 sums or fewer; B h sums `rank`
        products of h and the scale, in a chain; one more rounding adds the base."""
        y, tol = self.base[i].astype(np.float64), np.zeros((self.t, self.rows[i]))
        at = 0
        for n, a in zip(self.new, self.which):
            if 0 <= a < len(self.w[i]) and self.w[i][a] is not None:
                A, B, scale = self.w[i][a]
                x = self.x[at:at + n].astype(np.float64)
                h, hs = x @ A.T, np.abs(x) @ np.abs(A).T
                dh = (self.cols / 4 + 64) * U * hs
                y[at:at + n] += scale * (h @ B.T)
                tol[at:at + n] = abs(scale) * (dh @ np.abs(B).T + (A.shape[0] + 4) * U * (np.abs(h) @ np.abs(B).T))
            at += n
        tol += 2 * U * np.abs(y) + 1e-37
        tol[at:] = 0
        return y, tol

    def run(self, in_place=False, **kw):
        dx = dev(self.x)
        base = [dev(b) for b in self.base]
        y = base if in_place else [torch.full_like(b, 7.0) for b in base]
        torch.cuda.synchronize()
        apply_dev(self.sets, self.batch, dx.data_ptr(), [t.data_ptr() for t in y],
                  base_ptrs=None if in_place else [b.data_ptr() for b in base], **kw)
        wv.sync(kw.get("stream"))
        return [t.cpu().numpy() for t in y]

    def check(self, got, in_place=False):
        n = sum(self.new)
        for i, y in enumerate(got):
            want, tol = self.want(i)
            bad = ~(np.abs(y[:n].astype(np.float64) - want[:n]) <= tol[:n])
            assert not bad.any(), f"set {i}: {bad.sum()} values, off by {np.nanmax(np.abs(y[:n] - want[:n]))}"
            assert np.array_equal(y[n:], self.base[i][n:] if in_place else np.full_like(y[n:], 7.0)), "padding rows"
            at = 0
            for k, a in zip(self.new, self.which):
                if not (0 <= a < len(self.w[i]) and self.w[i][a] is not None):
                    assert np.array_equal(y[at:at + k], self.base[i][at:at + k])
                at += k


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("rows,cols,ranks,new,which", [
    (64, 64, [8], [1], [0]),
    (1, 1, [1], [1], [0]),
    (77, 61, [3, 17], [1, 1, 2], [1, 0, 1]),
    (300, 520, [16, 4, 0], [1] * 9, [0, 1, -1, 0, 2, 99, 1, 0, 0]),
    (1024, 4096, [32, 16], [1] * 64, [0, 1] * 32),
    (130, 1000, [64], [33], [0]),
    (257, 511, [20, 128], [100, 1, 0, 7, 32], [0, 1, 0, -1, 1]),
    (96, 5000, [256, 1], [5, 31, 64], [0, 1, 0]),
    (4100, 200, [48], [200, 3], [0, 0]),
    (33, 14336, [16], [4, 65], [0, 0]),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_sizes(typ, rows, cols, ranks, new, which, in_place):
    c = Case(np.random.default_rng(rows + cols), [rows], cols, ranks, new, which, typ, pad=2)
    c.check(c.run(in_place), in_place)


@pytest.mark.parametrize("new,which", [([1] * 5, [0, 1, 2, -1, 0]), ([40, 1, 90], [2, 0, 1])])
@pytest.mark.parametrize("ranks", [[16, 8, 30], [16, 3, 1], [80, 70, 2]])
@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_several_sets(new, which, ranks, typ):
    """Q, K and V: sets of unlike rows over the same input, and four at once; 48 to 320 ranks together."""
    rng = np.random.default_rng(3)
    for sets in ([512, 128, 128], [31, 700, 64, 5]):
        c = Case(rng, sets, 768, ranks, new, which, typ, pad=1)
        c.check(c.run())
        c.check(c.run(True), True)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("seqs,cols,hint", [(3, 700, 0), (300, 1100, 0), (300, 1100, 4), (5, 2500, 1)])
def test_short_sequences(n, seqs, cols, hint):
    """A few rows each, beside empty sequences: one range of the columns a block, or several."""
    rng = np.random.default_rng(n)
    c = Case(rng, [40, 9, 270], cols, [16, 40, 3], [0 if b % 7 == 3 else max(1, n - b % 3) for b in range(seqs)],
             [b % 4 - 1 for b in range(seqs)], pad=1)
    if hint:
        c.batch = AdapterBatch(seqs, c.t, c.cu.data_ptr(), c.ids.data_ptr(), hint)
    c.check(c.run())
    c.check(c.run(True), True)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("seqs,sets,cols,ranks,most", [
    (256, [300], 1500, [64, 40, 64], 1), (1000, [200, 33], 260, [16], 1), (1024, [70, 160, 40], 200, [16, 3, 0, 9], 2),
    (257, [1030], 700, [80] * 60, 4), (300, [96, 64], 1000, [48, 20, 33, 5, 1], 3),
])
def test_many_requests(seqs, sets, cols, ranks, most, typ):
    """Requests enough that those with one adapter are taken together: scattered, of no rows, without an adapter, of more
    rows than one tile, of more than the call is told of."""
    rng = np.random.default_rng(seqs)
    new = [0 if b % 11 == 5 else 1 + b % most for b in range(seqs)]
    which = list(rng.integers(-1, len(ranks) + 1, seqs))
    which[3:3 + seqs // 3] = [0] * (seqs // 3)
    if most > 2:
        new[7], new[-1] = 45, 90
    c = Case(rng, sets, cols, ranks, new, which, typ, pad=3)
    c.batch = AdapterBatch(seqs, c.t, c.cu.data_ptr(), c.ids.data_ptr(), most)
    got = c.run()
    c.check(got)
    assert all(np.array_equal(a, b) for a, b in zip(got, c.run()))
    c.check(c.run(True), True)


def test_many_requests_of_unlike_sets():
    """Sets of one call with more or fewer adapters than the requests name, at strides of their own."""
    rng = np.random.default_rng(12)
    which = [b % 40 for b in range(400)]
    a = Case(rng, [290], 500, [32] * 3, [1] * 400, which)
    b = Case(rng, [110], 500, [48] * 37, [1] * 400, which)
    x, base = dev(np.pad(a.x, ((0, 0), (0, 7)))), dev(rng.standard_normal((400, 600)).astype(np.float32))
    y = torch.full((400, 500), 7.0, device="cuda")
    torch.cuda.synchronize()
    c = AdapterBatch(400, 400, a.cu.data_ptr(), a.ids.data_ptr(), 1)
    apply_dev([a.sets[0], b.sets[0]], c, x.data_ptr(), [y.data_ptr(), y.data_ptr() + 4 * 301],
              base_ptrs=[base.data_ptr(), base.data_ptr() + 4 * 450], x_stride=507, y_strides=[500, 500],
              base_strides=[600, 600])
    wv.sync()
    h, got = base.cpu().numpy(), y.cpu().numpy()
    a.base, b.base, b.x = [h[:, :290]], [h[:, 450:560]], a.x
    for case, part in ((a, got[:, :290]), (b, got[:, 301:411])):
        want, tol = case.want(0)
        assert (np.abs(part - want) <= tol).all()
    assert (got[:, 290:301] == 7).all() and (got[:, 411:] == 7).all()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("new", [[10], [100] * 4, [300] * 4, [10, 2, 1, 4]])
def test_many_ranks(new, typ):
    """The sets' ranks by one block after another, by blocks of their own, or both."""
    c = Case(np.random.default_rng(len(new)), [130, 90], 2048, [128, 100], new, [b % 2 for b in range(len(new))], typ)
    c.check(c.run())


def test_sets_that_know_other_adapters():
    """Sets of one call with more or fewer adapters, of other ranks, some of them unset."""
    rng = np.random.default_rng(8)
    for new in ([1, 2, 1, 1], [40, 33, 64, 5]):
        a = Case(rng, [90, 200], 300, [16, 0, 7], new, [0, 1, 2, 0])
        b = Case(rng, [60], 300, [40], new, [0, 1, 2, 0])
        a.sets, a.w, a.rows, a.base = a.sets + b.sets, a.w + b.w, a.rows + b.rows, a.base + b.base
        a.check(a.run())
        a.sets, a.w, a.rows, a.base = a.sets[::-1], a.w[::-1], a.rows[::-1], a.base[::-1]
        a.check(a.run(True), True)


@pytest.mark.parametrize("hint", [0, 1, 4, 5, 1000])
def test_hints_only_steer(hint):
    """Whatever the call is told of its longest sequence."""
    c = Case(np.random.default_rng(hint), [300, 40], 600, [16, 40], [1, 70, 3, 0, 33], [0, 1, -1, 0, 0], pad=1)
    c.batch = AdapterBatch(5, c.t, c.cu.data_ptr(), c.ids.data_ptr(), hint)
    c.check(c.run())
    c.check(c.run(True), True)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_every_column_and_rank(n):
    """Tokens that are one column each: y is that column of A through B, within the roundings of one product chain."""
    rng = np.random.default_rng(n)
    cols, rank, rows = 700, 24, 50
    for first in range(0, cols, 100 * n if n < 40 else 40):
        c = Case(rng, [rows], cols, [rank], [n], [0])
        c.x[:] = 0
        at = (first + 17 * np.arange(n)) % cols
        c.x[np.arange(n), at] = rng.uniform(1, 2, n)
        c.base[0][:] = 0
        y = c.run()[0].astype(np.float64)
        A, B, scale = c.w[0][0]
        h = c.x[np.arange(n), at].astype(np.float64)[:, None] * A[:, at].T
        tol = scale * ((rank + 6) * U * (np.abs(h) @ np.abs(B).T)) + 1e-37
        assert (np.abs(y - scale * (h @ B.T)) <= tol).all()


@pytest.mark.parametrize("n", [1, 2, 50])
def test_strides_and_alignment(n):
    """Rows inside wider ones, at any multiple of 4 bytes, base and y at strides of their own."""
    rng = np.random.default_rng(11 + n)
    for off in (1, 2, 3):
        c = Case(rng, [70, 33], 130, [12], [n, 2], [0, 0])
        t = c.t
        fx = np.zeros(t * 137 + 4, np.float32)
        vx = fx[off:off + t * 137].reshape(t, 137)
        vx[:, :130] = c.x
        vx[:, 130:] = np.nan  # never read
        dx = dev(fx)
        bases, ys = [], []
        for i, (o, s) in enumerate(((70, 75), (33, 40))):
            b = np.zeros(t * s + 4, np.float32)
            b[off:off + t * s].reshape(t, s)[:, :o] = c.base[i]
            bases.append(dev(b))
            ys.append(torch.full((t * (s + 1) + 4,), 7.0, device="cuda"))
        torch.cuda.synchronize()
        apply_dev(c.sets, c.batch, dx.data_ptr() + 4 * off, [y.data_ptr() + 4 * off for y in ys],
                  base_ptrs=[b.data_ptr() + 4 * off for b in bases], x_stride=137, y_strides=[76, 41],
                  base_strides=[75, 40])
        wv.sync()
        got = []
        for y, (o, s) in zip(ys, ((70, 76), (33, 41))):
            y = y.cpu().numpy()
            rows = y[off:off + t * s].reshape(t, s)
            assert (rows[:, o:] == 7.0).all() and (y[:off] == 7.0).all() and (y[off + t * s:] == 7.0).all()
            got.append(rows[:, :o])
        c.check(got)


@pytest.mark.parametrize("new", [[1] * 4, [40, 2, 40, 33]])
def test_special_values_stay_in_their_rows(new):
    """NaN and infinity in one token's input: its own rows alone, and only through the adapter's own ranks."""
    c = Case(np.random.default_rng(9), [64], 256, [5, 16], new, [0, 1, -1, 0], max_rank=16)
    clean = c.run()[0]
    at = np.concatenate([[0], np.cumsum(new)])
    c.x[at[1], 100] = np.nan
    c.x[at[2], 3] = np.inf  # a sequence without an adapter
    c.x[at[3] + new[3] - 1, 255] = np.inf
    got = c.run()[0]
    hit = np.zeros(c.t, bool)
    hit[[at[1], at[3] + new[3] - 1]] = True
    assert np.array_equal(got[~hit], clean[~hit])
    assert np.isnan(got[at[1]]).all() and not np.isfinite(got[at[3] + new[3] - 1]).any()


def test_set_again_and_unset():
    rng = np.random.default_rng(21)
    c = Case(rng, [40], 90, [16, 16], [1, 1, 36], [0, 1, 0])
    c.check(c.run())
    a, av = held(rng.standard_normal((3, 90)) * 0.2, "bf16")
    b, bv = held(rng.standard_normal((40, 3)), "bf16")
    c.sets[0].set(0, a, b, -1.5)
    c.w[0][0] = (av, bv, -1.5)
    c.check(c.run())
    c.sets[0].unset(0)
    got = c.run()[0]
    assert np.array_equal(got[0], c.base[0][0]) and np.array_equal(got[2:], c.base[0][2:])


def test_streams_scratch_and_repeats():
    """A stream of one's own, scratch of one's own, the same bits every time."""
    c = Case(np.random.default_rng(5), [200, 64], 900, [32, 8], [1, 70, 1, 5], [0, 1, -1, 1], pad=1)
    first = c.run()
    c.check(first)
    s = torch.cuda.Stream()
    nb = scratch(c.sets, c.batch)
    sc = torch.full((nb // 4 + 4,), float("nan"), device="cuda")
    torch.cuda.synchronize()
    again = c.run(stream=s.cuda_stream, scratch_ptr=sc.data_ptr(), scratch_bytes=nb)
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    assert torch.isnan(sc[nb // 4:]).all()
    for code, text, kw in ((-2, "of scratch, needs", dict(scratch_ptr=sc.data_ptr(), scratch_bytes=nb - 4)),
                           (-1, "16-byte", dict(scratch_ptr=sc.data_ptr() + 4, scratch_bytes=nb))):
        with pytest.raises(wv.WelvetError) as e:
            c.run(**kw)
        assert e.value.code == code and text in str(e.value)


def test_captured():
    """A graph takes new rows, lengths and adapters on replay; without scratch of its own it is refused."""
    c = Case(np.random.default_rng(6), [150], 300, [16, 8], [1, 1, 34], [0, 1, 0])
    x, base = dev(c.x), dev(c.base[0])
    y = torch.zeros_like(base)
    nb = scratch(c.sets, c.batch)
    sc = torch.zeros(nb // 4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h = torch.cuda.current_stream().cuda_stream
        with pytest.raises(wv.WelvetError) as e:
            apply_dev(c.sets, c.batch, x.data_ptr(), [y.data_ptr()], base_ptrs=[base.data_ptr()], stream=h)
        assert e.value.code == -1 and "captured" in str(e.value)
        apply_dev(c.sets, c.batch, x.data_ptr(), [y.data_ptr()], base_ptrs=[base.data_ptr()], stream=h,
                  scratch_ptr=sc.data_ptr(), scratch_bytes=nb)
    for step, (new, which) in enumerate((([1, 1, 34], [0, 1, 0]), ([30, 5, 1], [1, -1, 0]), ([0, 36, 0], [0, 0, 1]))):
        c.new, c.which = new, which
        c.cu.copy_(dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)))
        c.ids.copy_(dev(np.array(which, np.int32)))
        c.x = np.random.default_rng(step).standard_normal(c.x.shape).astype(np.float32)
        x.copy_(dev(c.x))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager = c.run()  # the program's own call in between
        c.check([y.cpu().numpy()])
        c.check(eager)


def test_refusals():
    c = Case(np.random.default_rng(1), [64, 32], 96, [8], [2], [0])
    other = Case(np.random.default_rng(1), [64], 128, [8], [2], [0])
    half = Case(np.random.default_rng(1), [64], 96, [8], [2], [0], "f16")
    x, y = dev(c.x), [dev(b) for b in c.base]
    p = [t.data_ptr() for t in y]

    def call(sets=c.sets, batch=c.batch, xp=x.data_ptr(), yp=None, **kw):
        yp = (p if yp is None else yp)[: len(sets)]
        apply_dev(sets, batch, xp, yp + p[:1] * (len(sets) - len(yp)), **kw)

    q = c.cu.data_ptr()
    for code, text, fn in ((-2, "sets of", lambda: call([c.sets[0], other.sets[0]])),
                           (-2, "sets of", lambda: call([c.sets[0], half.sets[0]])),
                           (-2, "5 sets", lambda: call(c.sets[:1] * 5)),
                           (-2, "under the row", lambda: call(x_stride=95)),
                           (-2, "under the row", lambda: call(y_strides=[63, 32])),
                           (-2, "under the row", lambda: call(base_ptrs=p, base_strides=[64, 31])),
                           (-2, "base is y", lambda: call(base_ptrs=p, base_strides=[65, 32])),
                           (-1, "nil y", lambda: call(yp=[p[0], 0])),
                           (-1, "nil x", lambda: call(xp=0)),
                           (-1, "nil x", lambda: call(batch=AdapterBatch(1, 2, 0, q))),
                           (-1, "nil x", lambda: call(batch=AdapterBatch(1, 2, q, 0))),
                           (-2, "tokens", lambda: call(batch=AdapterBatch(1, 65536, q, q))),
                           (-2, "tokens", lambda: call(batch=AdapterBatch(-1, 2, q, q))),
                           (-1, "adapter 1 of 1", lambda: c.sets[0].set(1, *[np.zeros(s, np.uint16) for s in ((8, 96), (64, 8))])),
                           (-2, "rank 9", lambda: c.sets[0].set(0, *[np.zeros(s, np.uint16) for s in ((9, 96), (64, 9))])),
                           (-1, "scale", lambda: c.sets[0].set(0, *[np.zeros(s, np.uint16) for s in ((8, 96), (64, 8))],
                                                               float("inf")))):
        with pytest.raises(wv.WelvetError) as e:
            fn()
        assert e.value.code == code and text in str(e.value), str(e.value)
    call(batch=AdapterBatch(0, 0, 0, 0))
    call(batch=AdapterBatch(0, 2, 0, 0))
    wv.sync()
    for t, b in zip(y, c.base):
        assert np.array_equal(t.cpu().numpy(), b)
