"""Low-rank adapters on rows of all magnitudes, by tiles and by short sequences: each row within the roundings of its
own values, however small or large beside the others'."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from test_gpu_adapters import U, Case, dev, held
from welvet_amd.adapters import AdapterBatch, apply_dev

pytestmark = pytest.mark.gpu
TYPES = ["f16", "bf16"]


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def bound(x, A, B, scale, typ):
    """y without base, and what it may be off by. f32 products: chains of a quarter of the columns (or 16), joined by
    at most 40 sums, as in test_gpu_adapters. fp16 sets hold a tile's x and h as two fp16 terms under a power of two
    that brings the row's largest to 2^14: a value is off by 2^-22 of itself, or, where the second term is subnormal, by
    half of 2^-24 of those units, 2^-39 of the row's largest. bf16 sets hold them as three terms, exact but for what lies
    under the smallest subnormal: off by 2^-133. Sums below the normal f32 numbers are off by 2^-149."""
    x = x.astype(np.float64)
    top = np.abs(x).max(1, keepdims=True)
    h, hs = x @ A.T, np.abs(x) @ np.abs(A).T
    dh = (x.shape[1] / 4 + 64) * U * hs
    two = typ == "f16"
    dh += (2.0 ** -22 * hs + 2.0 ** -39 * top * np.abs(A).sum(1)) if two else 2.0 ** -133 * np.abs(A).sum(1)
    dh += 2.0 ** -148
    y, dy = scale * (h @ B.T), dh @ np.abs(B).T + (A.shape[0] + 4) * U * (np.abs(h) @ np.abs(B).T)
    dy *= abs(scale)
    if two:
        dy += abs(scale) * (2.0 ** -22 * (np.abs(h) @ np.abs(B).T)
                            + 2.0 ** -39 * (np.abs(h) + dh).max(1, keepdims=True) * np.abs(B).sum(1))
    else:
        dy += 2.0 ** -133 * np.abs(B).sum(1)  # h has its scale by then
    return y, dy + 2.0 ** -148 + 2 * U * np.abs(y)


def run(typ, x, new, scale, cols, rows=70, rank=20):
    rng = np.random.default_rng(cols)
    c = Case(rng, [rows], cols, [rank], new, [0] * len(new), typ)
    a, A = held(rng.standard_normal((rank, cols)) / np.sqrt(cols), typ)
    b, B = held(rng.standard_normal((rows, rank)) * 0.4, typ)
    c.sets[0].set(0, a, b, scale)
    c.x = x.astype(np.float32)
    c.base[0][:] = 0
    got = c.run()[0].astype(np.float64)
    want, tol = bound(c.x, A, B, float(np.float32(scale)), typ)
    assert np.isfinite(got).all()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{typ} rows {sorted(set(np.nonzero(bad)[0]))[:8]}: off by {np.abs(got - want)[bad].max()}" \
                          f" where {np.abs(want)[bad].max()}"


SIZES = [2.0 ** -110, 2.0 ** -111, 2.0 ** -112, 2.0 ** -113, 2.0 ** -114, 1e-36, 1e-30, 1e-12, 1.0, 1e12, 1e30]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("new", [[40, 33], [5] * 15, [1] * 66, [3] * 22])
@pytest.mark.parametrize("cols", [61, 1100])
def test_rows_of_one_magnitude(typ, new, cols):
    """All rows alike, with a scale that brings the small ones back."""
    rng = np.random.default_rng(sum(new))
    x = rng.uniform(0.5, 1.0, (sum(new), cols)) * rng.choice([-1, 1], (sum(new), cols))
    for size in SIZES:
        run(typ, x * size, new, 1 / size if 1e-37 < size else 2.0 ** 100, cols)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("new", [[66], [5] * 14, [2] * 33])
def test_rows_of_unlike_magnitudes(typ, new):
    """Side by side in a tile."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((sum(new), 500)) * np.array(SIZES)[np.arange(sum(new)) % len(SIZES)][:, None]
    run(typ, x, new, 1.0, 500)
    x = x * (np.abs(x).max(1, keepdims=True) < 1e-20) * 2.0 ** -3  # the others' results would be past f32
    run(typ, x, new, 2.0 ** 100, 500)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("up", [False, True])
def test_columns_of_unlike_magnitudes(typ, up):
    """Within a row: growing or falling along it, over a range that the sums' units have to follow."""
    rng = np.random.default_rng(4)
    e = np.linspace(-115, 60, 2048) if up else np.linspace(60, -115, 2048)
    x = rng.uniform(0.5, 1.0, (40, 2048)) * 2.0 ** np.round(e)
    run(typ, x, [40], 1.0, 2048)
    x[:, : 1024] = 0  # only the small, or only the large half
    run(typ, x, [40], 1.0, 2048)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n", [3, 40])
def test_single_columns(typ, n):
    """Tokens that are one column each: y is that column of A through B, within the roundings of one product chain and,
    by tiles, of x and h as `bound` has them."""
    rng = np.random.default_rng(n)
    cols, rank, rows = 700, 24, 50
    for size in (1.0, 2.0 ** -112, 1e-36, 1e30):
        c = Case(rng, [rows], cols, [rank], [n], [0], typ)
        A, B, _ = c.w[0][0]
        scale = float(np.float32(2.0 ** 100 if size < 1e-30 else 1.0))
        c.sets[0].set(0, held(A, typ)[0], held(B, typ)[0], scale)
        for first in range(0, cols, 40 if n == 40 else 100):
            c.x[:] = 0
            at = (first + 17 * np.arange(n)) % cols
            c.x[np.arange(n), at] = rng.uniform(1, 2, n) * size
            c.base[0][:] = 0
            y = c.run()[0].astype(np.float64)
            h = c.x[np.arange(n), at].astype(np.float64)[:, None] * A[:, at].T
            s = np.abs(h) @ np.abs(B).T
            tol = scale * (rank + 6) * U * s + 2.0 ** -148
            if typ == "f16":
                tol += scale * (2.0 ** -21 * s + 2.0 ** -38 * np.abs(h).max(1, keepdims=True) * np.abs(B).sum(1))
            else:
                tol += 2.0 ** -133 * (scale * np.abs(A[:, at].T) + 1) @ np.abs(B).T
            assert (np.abs(y - scale * (h @ B.T)) <= tol).all(), f"{typ}, {size}, column {first} on"


@pytest.mark.parametrize("typ", TYPES)
def test_small_rows_by_adapter(typ):
    """Requests enough that their rows are taken by adapter."""
    rng = np.random.default_rng(9)
    n, cols, rows = 600, 1500, 300
    c = Case(rng, [rows], cols, [64, 40], [1] * n, [b % 2 for b in range(n)], typ)
    size = np.array(SIZES)[np.arange(n) // 2 % len(SIZES)][:, None]
    c.x = (rng.standard_normal((n, cols)) * size).astype(np.float32)
    base = torch.zeros(n, rows, device="cuda")
    x = dev(c.x)
    w = []
    for j in range(2):
        A, B, _ = c.w[0][j]
        c.sets[0].set(j, held(A, typ)[0], held(B, typ)[0], 2.0 ** 20)
        w.append((A, B))
    b = AdapterBatch(n, n, c.cu.data_ptr(), c.ids.data_ptr(), 1)
    apply_dev(c.sets, b, x.data_ptr(), [base.data_ptr()])
    wv.sync()
    y = base.cpu().numpy().astype(np.float64)
    for j in range(2):
        want, tol = bound(c.x[j::2], *w[j], 2.0 ** 20, typ)
        assert (np.abs(y[j::2] - want) <= tol).all()
