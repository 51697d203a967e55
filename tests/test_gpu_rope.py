"""Rotary positions on the device against the same rotation in float64."""
import math

import numpy as np
import pytest
import torch

import welvet_amd as wv
from welvet_amd.rope import Rope

pytestmark = pytest.mark.gpu

# An angle is off by 2^-26 of a turn (its fraction in f32), 9.4e-8; sine and cosine by 2 steps of 2^-24 each,
# together 1.7e-7; gain and its products by 2^-23; the two products and their sum by 2^-23: 5e-7 of gain times the
# pair's length.
TOL = 6e-7


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def freqs(rot, theta, scaling="none", factor=1.0, trained=0, low=1.0, high=32.0):
    i = np.arange(rot // 2)
    if scaling == "base":
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "ramp_turns":
        r = (trained * f / (2 * math.pi) - low) / (high - low)
    elif scaling == "ramp_dims":
        at = lambda n: rot * math.log(trained / (2 * math.pi * n)) / (2 * math.log(theta))  # noqa: E731
        i0, i1 = (min(max(x, 0), rot // 2 - 1) for x in (math.floor(at(high)), math.ceil(at(low))))
        r = 1 - (i - i0) / max(i1 - i0, 0.001)
    else:
        return f
    r = np.clip(r, 0, 1)
    return f / factor * (1 - r) + f * r


def turned(x, pos, f, layout, rot, gain):
    """x [n, heads, hd] in f64, and gain times the length of each value's pair."""
    x = x.astype(np.float64)
    t = pos.astype(np.float64)[:, None] * f
    c, s = (fn(t)[:, None] * gain for fn in (np.cos, np.sin))
    y, size = x.copy(), np.zeros_like(x)
    a = np.arange(rot // 2) if layout == "half" else 2 * np.arange(rot // 2)
    b = a + (rot // 2 if layout == "half" else 1)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = np.hypot(x[..., a], x[..., b]) * gain
    return y, size


def dev(x):
    d = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    torch.cuda.synchronize()
    return d


def check(got, x, pos, f, layout, rot, gain, tol=TOL):
    y, size = turned(x, pos, f, layout, rot, gain)
    d = np.abs(got.astype(np.float64) - y)
    assert (d <= tol * size + 1e-37).all(), f"off by {np.max(d - tol * size)}"
    assert np.array_equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("hd,rot,n,heads,kv", [(128, 128, 1, 32, 8), (64, 64, 5, 7, 1), (80, 20, 33, 3, 2), (2, 2, 3, 1, 1),
                                               (256, 128, 17, 4, 4), (6, 4, 40, 5, 0), (1024, 1022, 3, 2, 1),
                                               (128, 64, 300, 8, 8), (66, 66, 9, 2, 3),
                                               (80, 22, 30, 5, 2), (8, 2, 600, 300, 1), (64, 60, 5, 70, 3)])
def test_layouts(layout, hd, rot, n, heads, kv):
    rng = np.random.default_rng(hd + rot + n)
    r = Rope(hd, rot, theta=1e4, layout=layout)
    q, k = (rng.standard_normal((n, h, hd)).astype(np.float32) for h in (heads, kv))
    pos = rng.integers(0, 5000, n).astype(np.int32)
    dq, dk, dp = dev(q), dev(k), dev(pos)
    r.apply_dev(dp.data_ptr(), n, dq.data_ptr(), heads, dk.data_ptr() or None, kv)
    wv.sync()
    for d, x in ((dq, q), (dk, k)):
        check(d.cpu().numpy(), x, pos, freqs(rot, 1e4), layout, rot, 1.0)


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "ramp_dims", "ramp_turns"])
@pytest.mark.parametrize("factor,trained,gain", [(8.0, 8192, 1.0), (2.5, 500, 1.2079), (0.5, 100000, 0.7)])
def test_scaled(scaling, factor, trained, gain):
    rng = np.random.default_rng(7)
    kw = dict(scaling=scaling, factor=factor, trained=trained, low=1.0, high=32.0)
    r = Rope(128, 96, theta=5e5, layout="half", gain=gain, **kw)
    x = rng.standard_normal((64, 4, 128)).astype(np.float32)
    pos = np.concatenate([rng.integers(0, 1 << 20, 62), [0, 1]]).astype(np.int32)
    d, p = dev(x), dev(pos)
    r.apply_dev(p.data_ptr(), 64, d.data_ptr(), 4)
    wv.sync()
    check(d.cpu().numpy(), x, pos, freqs(96, 5e5, **kw), "half", 96, gain)


def test_far_positions():
    """Positions up to the largest: there a turn of f64 is 2^-22 fine, and the frequencies themselves count."""
    x = np.random.default_rng(2).standard_normal((6, 2, 64)).astype(np.float32)
    pos = np.array([1 << 24, (1 << 24) - 1, -(1 << 24), (1 << 31) - 1, -(1 << 31), 0], np.int64).astype(np.int32)
    d, p = dev(x), dev(pos)
    Rope(64, theta=1e4).apply_dev(p.data_ptr(), 6, d.data_ptr(), 2)
    wv.sync()
    got = d.cpu().numpy()
    check(got[[0, 1, 2, 5]], x[[0, 1, 2, 5]], pos[[0, 1, 2, 5]], freqs(64, 1e4), "half", 64, 1.0)
    check(got[3:5], x[3:5], pos[3:5], freqs(64, 1e4), "half", 64, 1.0, tol=2e-6)


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_strides_and_outputs(layout, off):
    """Rows inside wider ones at any multiple of 4 bytes, with outputs of their own; what lies between stays."""
    n, heads, kv, hd, rot = 9, 6, 2, 64, 48
    rng = np.random.default_rng(off)
    w = (heads + 2 * kv) * hd + 5  # q | k | v rows
    x = rng.standard_normal((n, w)).astype(np.float32)
    pos = rng.integers(0, 900, n).astype(np.int32)
    flat = np.zeros(n * w + 8, np.float32)
    flat[off:off + n * w] = x.reshape(-1)
    d, p = dev(flat), dev(pos)
    qo = torch.full((n * (heads * hd + 3) + 8,), 7.0, device="cuda")
    ko = torch.full((n, kv * hd), 7.0, device="cuda")
    torch.cuda.synchronize()
    r = Rope(hd, rot, theta=1e4, layout=layout, gain=1.5)
    base = d.data_ptr() + 4 * off
    r.apply_dev(p.data_ptr(), n, base, heads, base + 4 * heads * hd, kv, q_stride=w, k_stride=w,
                q_out_ptr=qo.data_ptr() + 4 * off, k_out_ptr=ko.data_ptr(), q_out_stride=heads * hd + 3)
    wv.sync()
    assert np.array_equal(d.cpu().numpy(), flat)
    got = qo.cpu().numpy()
    rows = got[off:off + n * (heads * hd + 3)].reshape(n, -1)
    assert (rows[:, heads * hd:] == 7.0).all() and (got[:off] == 7.0).all() and (got[off + rows.size:] == 7.0).all()
    f = freqs(rot, 1e4)
    check(rows[:, : heads * hd].reshape(n, heads, hd), x[:, : heads * hd].reshape(n, heads, hd), pos, f, layout, rot, 1.5)
    check(ko.cpu().numpy().reshape(n, kv, hd), x[:, heads * hd:(heads + kv) * hd].reshape(n, kv, hd), pos, f, layout, rot,
          1.5)
    r.apply_dev(p.data_ptr(), n, base, heads, base + 4 * heads * hd, kv, q_stride=w, k_stride=w)  # in place
    wv.sync()
    after = d.cpu().numpy()[off:off + n * w].reshape(n, w)
    assert np.array_equal(after[:, : heads * hd], rows[:, : heads * hd])
    assert np.array_equal(after[:, heads * hd:(heads + kv) * hd], ko.cpu().numpy())
    assert np.array_equal(after[:, (heads + kv) * hd:], x[:, (heads + kv) * hd:])


def test_gradient():
    """The rotation is linear: its gradient is the call at the negative position, as differences of the call say too."""
    rng = np.random.default_rng(4)
    n, heads, hd, rot, gain = 3, 2, 64, 32, 1.25
    r = Rope(hd, rot, theta=1e4, gain=gain)
    x, g = (rng.standard_normal((n, heads, hd)).astype(np.float32) for _ in range(2))
    pos = np.array([5, 1000, 70001], np.int32)

    def call(v, p):
        d, q = dev(v.astype(np.float32)), dev(p)
        r.apply_dev(q.data_ptr(), n, d.data_ptr(), heads)
        wv.sync()
        return d.cpu().numpy().astype(np.float64)

    grad = call(g, -pos)
    for _ in range(4):
        u = rng.standard_normal(x.shape).astype(np.float32)
        # linear, so a difference of any width is exact but for rounding: each side is a sum of 384 products off by
        # TOL of the pairs' lengths
        up, down = (x + u).astype(np.float32), (x - u).astype(np.float32)
        diff = ((call(up, pos) - call(down, pos)) * g).sum()
        want = (grad * (up.astype(np.float64) - down)).sum()
        size = (np.abs(grad).max() * np.abs(up - down).max() * x.size)
        assert abs(diff - want) <= 4 * TOL * size


def test_special_values_and_none():
    """A NaN or infinity reaches its own pair alone; no rows, no heads."""
    x = np.ones((2, 1, 8), np.float32)
    x[0, 0, 1], x[1, 0, 7] = np.nan, np.inf
    d, p = dev(x), dev(np.array([3, 0], np.int32))
    r = Rope(8, 6, theta=100.0)
    r.apply_dev(p.data_ptr(), 2, d.data_ptr(), 1)
    wv.sync()
    got = d.cpu().numpy()
    assert np.isnan(got[0, 0, [1, 4]]).all() and np.isfinite(got[0, 0, [0, 2, 3, 5, 6, 7]]).all()
    assert np.isinf(got[1, 0, 7]) and np.array_equal(got[1, 0, :7], np.ones(7, np.float32))
    r.apply_dev(p.data_ptr(), 0, d.data_ptr(), 1)
    r.apply_dev(p.data_ptr(), 2)
    wv.sync()
    assert np.array_equal(d.cpu().numpy(), got, equal_nan=True)


def test_captured():
    r = Rope(64, theta=1e4)
    x = dev(np.random.default_rng(1).standard_normal((4, 2, 64)).astype(np.float32))
    y, p = torch.zeros_like(x), dev(np.zeros(4, np.int32))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r.apply_dev(p.data_ptr(), 4, x.data_ptr(), 2, q_out_ptr=y.data_ptr(),
                    stream=torch.cuda.current_stream().cuda_stream)
    for step in range(3):
        pos = np.arange(4, dtype=np.int32) * 100 + step
        p.copy_(dev(pos))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(y.cpu().numpy(), x.cpu().numpy(), pos, freqs(64, 1e4), "half", 64, 1.0)


def test_refusals():
    r = Rope(64)
    x = dev(np.zeros((4, 2, 64), np.float32))
    p = dev(np.zeros(4, np.int32))
    a = x.data_ptr()
    for call, code, text in ((lambda: r.apply_dev(p.data_ptr(), -1, a, 2), -2, "rows"),
                             (lambda: r.apply_dev(p.data_ptr(), 4, a, -1), -2, "heads"),
                             (lambda: r.apply_dev(p.data_ptr(), 4, a, 65536), -2, "heads"),
                             (lambda: r.apply_dev(p.data_ptr(), 4, a, 2, q_stride=127), -2, "under the row"),
                             (lambda: r.apply_dev(p.data_ptr(), 4, a, 1, q_stride=128, q_out_ptr=a), -2, "in place"),
                             (lambda: r.apply_dev(p.data_ptr(), 4, None, 2), -1, "nil rows"),
                             (lambda: r.apply_dev(p.data_ptr(), 4, a, 2, None, 1), -1, "nil rows"),
                             (lambda: r.apply_dev(None, 4, a, 2), -1, "nil pos")):
        with pytest.raises(wv.WelvetError) as e:
            call()
        assert e.value.code == code and text in str(e.value)
    assert not x.cpu().numpy().any()


def test_rows_of_a_call():
    """2^23 rows a call: more are refused, before anything is read."""
    r = Rope(2, theta=1e4)
    x = dev(np.ones((1, 1, 2), np.float32))
    with pytest.raises(wv.WelvetError) as e:
        r.apply_dev(x.data_ptr(), (1 << 23) + 1, x.data_ptr(), 1)
    assert e.value.code == -2 and "at most 2^23" in str(e.value)
    n = 1 << 23
    pos = torch.arange(n, dtype=torch.int32, device="cuda") % 1000
    y = torch.ones(n, 1, 2, device="cuda")
    torch.cuda.synchronize()
    r.apply_dev(pos.data_ptr(), n, y.data_ptr(), 1)
    wv.sync()
    y = y.cpu().numpy()
    check(y[-5:], np.ones((5, 1, 2), np.float32), np.arange(n - 5, n) % 1000, freqs(2, 1e4), "half", 2, 1.0)
    assert np.array_equal(y[:n // 8 // 1000 * 1000].reshape(-1, 1000, 2)[::97], np.broadcast_to(
        y[:1000].reshape(1, 1000, 2), (len(range(0, n // 8 // 1000, 97)), 1000, 2)))
