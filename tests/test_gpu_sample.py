"""wv_sample_dev against the definition in float64: every setting alone and together, ties, masked and
non-finite logits, row strides, vocabularies from one token to 2^19, borders of u and of the cuts.

Weights on the device are off by a step of the f32 exponential and by the rounding of its argument a, 2^-24 |a|
ln 2, whose sign changes from token to token: weights down to 2^-5 by 2^-22 each, and sums of smaller ones, which
take many, by less. Sums are exact: a running sum over a total is off by 2^-21 (OFF). A draw has to be the reference's token, or one
that the reference gives when its borders (the sum at u, the top-p prefix, min_p) move by that much."""
import ctypes

import numpy as np
import pytest
import torch

import welvet_amd as wv
from welvet_amd.sampling import Sampling, sample_dev

pytestmark = pytest.mark.gpu
OFF = 2.0 ** -21


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def reference(l, t, k, p, m, u):
    """The drawn token and its share, and accepts(token): whether a draw that is off by OFF at its borders may
    give it. With the fewest (lo) and the most (hi) tokens that the cuts can keep, its running sums lie between
    those over lo and over hi, and so does u times the total."""
    l = np.where(np.isnan(l), -np.inf, np.asarray(l, np.float64))
    top = l.max()
    if top == -np.inf:
        return -1, 0.0, lambda i: i == -1
    if not t > 0 or k == 1 or p <= 0:
        best = int(np.argmax(l))
        return best, 1.0, lambda i: i == best
    order = np.lexsort((np.arange(l.size), -l))
    if 0 < k < l.size:
        order = order[:k]
    with np.errstate(all="ignore"):
        w = np.where(l[order] == top, 1.0, np.exp((l[order] - top) / np.float64(t)))
    w[(l[order] == -np.inf) | ((top == np.inf) & (l[order] != top))] = 0  # whatever the temperature
    m = min(m, 1.0) if m > 0 else 0.0
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24) if u == u else 0.0

    def sums(off):  # the kept weights by index, as off moves the cuts
        keep = w >= m * (1 + off if m < 1 else 1)
        if p < 1:
            mass = np.cumsum(w)
            n = int(np.searchsorted(mass, np.float64(p) * mass[-1] * (1 - off), side="left")) + 1
            keep &= np.arange(w.size) < n
        x = np.zeros(l.size)
        x[order] = w * keep
        return x, np.cumsum(x)

    (x, run), (_, lo), (xh, hi) = sums(0.0), sums(OFF), sums(-OFF)
    at = int(np.searchsorted(run, u * run[-1], side="right"))

    def accepts(i):
        return (0 <= i < l.size and xh[i] > 0 and (lo[i - 1] if i else 0.0) - OFF * hi[-1] <= u * hi[-1]
                and hi[i] + OFF * hi[-1] >= u * lo[-1])
    return at, x[at] / run[-1], accepts


def draw(l, t=None, k=None, p=None, m=None, u=None, pad=0, off=0, stream=None):
    r, v = l.shape
    buf = torch.full((off + r * (v + pad),), 1e30, device="cuda")
    view = buf[off:].view(r, v + pad)
    view[:, :v] = torch.from_numpy(np.ascontiguousarray(l))
    arr = [None if x is None else torch.from_numpy(np.broadcast_to(np.asarray(x, d), (r,)).copy()).cuda()
           for x, d in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32), (u, np.float32))]
    tok = torch.full((r + 1,), -9, dtype=torch.int32, device="cuda")
    prob = torch.full((r + 1,), -9.0, device="cuda")
    ptr = [None if x is None else x.data_ptr() for x in arr]
    torch.cuda.synchronize()
    sample_dev(view.data_ptr(), r, v, tok.data_ptr(), ptr[4], stride=v + pad, temperature_ptr=ptr[0],
               top_k_ptr=ptr[1], top_p_ptr=ptr[2], min_p_ptr=ptr[3], probs_ptr=prob.data_ptr(), stream=stream)
    wv.sync(stream)
    assert int(tok[r]) == -9 and float(prob[r]) == -9.0
    return tok[:r].cpu().numpy(), prob[:r].cpu().numpy()


def check(l, t=None, k=None, p=None, m=None, u=None, **kw):
    r = l.shape[0]
    tok, prob = draw(l, t, k, p, m, u, **kw)
    full = [np.broadcast_to(np.asarray(d if x is None else x, ty), (r,))
            for x, d, ty in ((t, 1, np.float32), (k, 0, np.int32), (p, 1, np.float32), (m, 0, np.float32),
                             (u, 0, np.float32))]
    same = 0
    for i in range(r):
        want, share, accepts = reference(l[i], *(x[i] for x in full))
        assert accepts(int(tok[i])), f"row {i}: {tok[i]}, want {want}"
        if tok[i] == want:
            same += 1
            # the total may differ by the tokens at the cuts' borders
            assert abs(prob[i] - share) <= 2.0 ** -19 * share + 2.0 ** -44, f"row {i}: {prob[i]}, want {share}"
    assert same >= 0.9 * r or r - same <= 1, f"{same} of {r} rows as the reference"
    return tok


def logits(rng, r, v, spread=2.5):
    return (rng.standard_normal((r, v)) * spread).astype(np.float32)


VOCABS = [1, 2, 63, 1000, 4097, 8192, 8193, 32000, 32768, 32769, 50001, 131072]
SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=40), dict(k=128), dict(k=129), dict(k=1500), dict(p=0.9),
            dict(p=0.1, t=1.5), dict(m=0.05), dict(k=50, p=0.95), dict(k=700, p=0.6, m=0.01), dict(t=0.0),
            dict(p=0.999, t=2.0), dict(k=64, m=1.0)]


@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("s", range(len(SETTINGS)))
def test_settings(v, s):
    rng = np.random.default_rng(v * 31 + s)
    r = 6
    check(logits(rng, r, v), u=rng.random(r, np.float32), pad=(0, 3)[s % 2], off=(0, 1)[s % 2],
          **SETTINGS[s])


def test_largest_vocab():
    rng = np.random.default_rng(2)
    for s in (dict(), dict(p=0.9), dict(k=300), dict(k=40, p=0.9)):
        check(logits(rng, 2, 1 << 19), u=rng.random(2, np.float32), **s)


def test_mixed_rows():
    """Every row its own settings, greedy ones among them."""
    rng = np.random.default_rng(3)
    r = 200
    check(logits(rng, r, 5000), t=rng.choice([0, 0.5, 1, 1.7], r), k=rng.choice([0, 1, 7, 50, 400, 9999], r),
          p=rng.choice([0.0, 0.3, 0.9, 1.0, 1.5], r), m=rng.choice([0, 0.1, 0.001], r), u=rng.random(r, np.float32))


@pytest.mark.parametrize("v", [70, 3000, 33000, 100000])
@pytest.mark.parametrize("s", [dict(k=5), dict(k=200), dict(p=0.25), dict(k=1200, p=0.5), dict(k=9, m=0.5)])
def test_all_equal(v, s):
    """One logit for all tokens: every cut falls among ties, which go by index."""
    u = np.array([0, 0.1, 0.49, 0.75, 0.999], np.float32)
    l = np.full((5, v), -3.25, np.float32)
    tok, prob = draw(l, u=u, **s)
    kept = v
    if 0 < s.get("k", 0) < v:
        kept = s["k"]
    if "p" in s:
        kept = int(np.ceil(np.float64(np.float32(s["p"])) * kept))
    assert np.array_equal(tok, np.floor(u.astype(np.float64) * kept).astype(int))
    assert np.allclose(prob, 1 / kept, rtol=2.0 ** -22, atol=0)


def test_few_levels():
    """Thousands of ties at each of a few logits, zeros of both signs among them."""
    rng = np.random.default_rng(4)
    l = rng.choice(np.array([1.0, 0.5, 0.0, -0.0, -2.0], np.float32), (12, 40000))
    u = rng.random(12, np.float32)
    for s in (dict(k=100), dict(k=20000), dict(p=0.8), dict(k=30000, p=0.7), dict(m=0.3)):
        check(l, u=u, **s)


def test_masked_and_non_finite():
    rng = np.random.default_rng(5)
    l = logits(rng, 8, 2000)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, :] = -np.inf
    l[2, 1234] = -80.0
    l[3, ::2] = -np.inf
    l[4, 5::7] = np.nan
    l[5, 77], l[5, 1300] = np.inf, np.inf
    l[6] *= np.float32(1e37)
    l[7, :1990] = -np.inf
    u = rng.random(8, np.float32)
    for s in (dict(), dict(k=50), dict(k=500), dict(p=0.9), dict(t=0.0), dict(k=30, p=0.5, m=0.1), dict(t=1e-30),
              dict(t=3e38), dict(t=np.inf)):
        tok = check(l, u=u, **s)
        assert tok[0] == -1 and tok[1] == -1 and tok[2] == 1234
        assert tok[3] % 2 == 1 and tok[4] % 7 != 5 and tok[5] in (77, 1300) and tok[7] >= 1990


@pytest.mark.parametrize("v", [70, 6000, 20000, 33000, 150000])
@pytest.mark.parametrize("s", [dict(k=40), dict(k=40, p=0.9), dict(k=500), dict(k=500, p=0.9), dict(p=0.9), dict()])
def test_few_unmasked(v, s):
    """Fewer tokens that are not -inf than top_k asks for, one alone among them."""
    rng = np.random.default_rng(v)
    l = np.full((7, v), -np.inf, np.float32)
    for r, n in enumerate((1, 2, 5, 17, 30, 39, 40)):
        at = rng.permutation(v)[:n]
        l[r, at] = logits(rng, 1, n)[0]
    check(l, t=0.9, u=rng.random(7, np.float32), **s)


def test_settings_out_of_range():
    rng = np.random.default_rng(6)
    l = logits(rng, 10, 777)
    l[:, 600] = 9.0
    best = l.argmax(1)
    u = np.array([-1, 0, 1, 2, np.nan, np.inf, -np.inf, 0.5, 0.9, 1 - 2.0 ** -24], np.float32)
    check(l, u=u)
    check(l, u=u, k=-5, p=np.nan, m=np.nan)
    check(l, u=u, m=-1.0, p=7.0)
    assert (check(l, u=u, m=5.0) == best).all()
    assert (check(l, u=u, t=np.nan) == best).all()
    assert (check(l, u=u, t=-1.0) == best).all()
    assert (check(l, u=u, p=-0.5) == best).all()


def test_distribution():
    """Draws over an even grid of u come as often as the weights say, to one grid step per token."""
    rng = np.random.default_rng(7)
    n = 4096
    one = logits(rng, 1, 50, 1.0)
    tok = draw(np.repeat(one, n, 0), t=0.8, u=(np.arange(n) + 0.5) / n)[0]
    w = np.exp((one[0].astype(np.float64) - one.max()) / np.float64(np.float32(0.8)))
    assert np.abs(np.bincount(tok, minlength=50) / n - w / w.sum()).max() <= 1.5 / n
    assert (np.diff(tok) >= 0).all()


def test_repeatable_and_replayed():
    """The same bits again, and from a captured call whose inputs change between replays."""
    rng = np.random.default_rng(8)
    r, v = 9, 40000
    l, t = torch.empty(r, v, device="cuda"), torch.full((r,), 0.9, device="cuda")
    p, u = torch.full((r,), 0.9, device="cuda"), torch.zeros(r, device="cuda")
    tok, prob = torch.zeros(r, dtype=torch.int32, device="cuda"), torch.zeros(r, device="cuda")
    st = torch.cuda.Stream()
    l.zero_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        sample_dev(l.data_ptr(), r, v, tok.data_ptr(), u.data_ptr(), temperature_ptr=t.data_ptr(),
                   top_p_ptr=p.data_ptr(), probs_ptr=prob.data_ptr(), stream=st.cuda_stream)
    for i in range(3):
        x, y = logits(rng, r, v), rng.random(r, np.float32)
        l.copy_(torch.from_numpy(x))
        u.copy_(torch.from_numpy(y))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        a, b = draw(x, t=0.9, p=0.9, u=y)
        assert np.array_equal(a, tok.cpu().numpy()) and np.array_equal(b, prob.cpu().numpy())
        check(x, t=0.9, p=0.9, u=y)


def test_many_rows_of_a_large_vocab():
    """More rows than are cut over blocks: each by one block that reads it from memory in every pass."""
    rng = np.random.default_rng(12)
    r, v = 131, 33001
    x = logits(rng, r, v)
    x[3] = -np.inf
    x[7, 5:] = x[7, 5]
    pick = lambda *a: rng.choice(np.array(a, np.float32), r)  # noqa: E731
    check(x, t=pick(0.0, 0.7, 1.0), k=pick(0, 1, 40, 500).astype(np.int32), p=pick(0.5, 0.95, 1.0),
          m=pick(0, 0.01), u=rng.random(r, np.float32))


def test_two_streams():
    """Calls on two streams at once, each with scratch of its own: the bits of calls one after the other."""
    rng = np.random.default_rng(13)
    v, st = 70000, [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for r in (17, 40):
        x, u = logits(rng, r, v), rng.random(r, np.float32)
        want = draw(x, t=0.9, p=0.9, u=u)
        sets.append((r, torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), torch.full((r,), 0.9, device="cuda"), want,
                     [torch.zeros(r, dtype=torch.int32, device="cuda") for _ in range(6)],
                     [torch.zeros(r, device="cuda") for _ in range(6)]))
    torch.cuda.synchronize()
    for i in range(6):
        for s, (r, x, u, a, _, tok, prob) in zip(st, sets):
            sample_dev(x.data_ptr(), r, v, tok[i].data_ptr(), u.data_ptr(), temperature_ptr=a.data_ptr(),
                       top_p_ptr=a.data_ptr(), probs_ptr=prob[i].data_ptr(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for r, _, _, _, want, tok, prob in sets:
        for i in range(6):
            assert np.array_equal(tok[i].cpu().numpy(), want[0]) and np.array_equal(prob[i].cpu().numpy(), want[1])


def test_no_probs_and_refusals():
    L = wv.lib()
    l, u = torch.zeros(2, 100, device="cuda"), torch.tensor([0.5, 0.995], device="cuda")
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sample_dev(l.data_ptr(), 2, 100, tok.data_ptr(), u.data_ptr())
    wv.sync()
    assert tok.tolist() == [50, 99]
    s = Sampling(None, None, None, None, u.data_ptr())
    by = ctypes.byref(s)
    P, T = l.data_ptr(), tok.data_ptr()
    assert L.wv_sample_dev(P, 0, 0, 100, by, T, None, None) == 0
    assert L.wv_sample_dev(P, 0, -1, 100, by, T, None, None) == -2
    assert L.wv_sample_dev(P, 0, 1, 0, by, T, None, None) == -2
    assert L.wv_sample_dev(P, 0, 1, (1 << 19) + 1, by, T, None, None) == -2
    assert L.wv_sample_dev(P, 99, 1, 100, by, T, None, None) == -2
    assert L.wv_sample_dev(None, 0, 1, 100, by, T, None, None) == -1
    assert L.wv_sample_dev(P, 0, 1, 100, by, None, None, None) == -1
    assert L.wv_sample_dev(P, 0, 1, 100, None, T, None, None) == -1
    s2 = Sampling(None, None, None, None, None)
    assert L.wv_sample_dev(P, 0, 1, 100, ctypes.byref(s2), T, None, None) == -1
