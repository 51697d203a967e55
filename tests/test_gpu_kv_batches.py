"""Attention over batches of more sequences than a wave looks at at once: ragged ones, idle ones, chunks behind the
64th and the 128th, for the row and the tile kernel."""
import numpy as np
import pytest

import welvet_amd as wv
from test_gpu_kv import Pool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def batch(rng, seqs, chunks, longest):
    """New tokens: one each, some idle, `chunks` {sequence: tokens}; and lengths that hold them."""
    new = [0 if i % 11 == 3 else 1 for i in range(seqs)]
    for i, n in chunks.items():
        new[i] = n
    return new, [int(max(n, rng.integers(1, longest))) for n in new]


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("seqs,chunks", [(65, {}), (65, {64: 70}), (130, {2: 9, 64: 33, 129: 120}), (200, {128: 5, 198: 64})])
@pytest.mark.parametrize("max_q", [0, 1, 128])
def test_row_kernel(typ, seqs, chunks, max_q):
    """max_q of 1 with a chunk in the batch: its later tiles are found behind the sequences' first ones."""
    rng = np.random.default_rng(seqs)
    new, lens = batch(rng, seqs, chunks, 200)
    p = Pool(rng, lens, 2, 64, 32, typ).fill()
    p.check(p.attend(new, 8, max_q=max_q, pad=2), new)
    p.check(p.attend(new, 8, max_q=max_q, window=40), new, window=40)


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 64), (32, 8, 128)])
def test_tile_kernel(typ, heads, kv_heads, hd):
    """Long chunks on either side of the 64th and 128th sequence beside single tokens."""
    rng = np.random.default_rng(hd)
    new, lens = batch(rng, 140, {1: 900, 63: 300, 64: 1200, 130: 1000, 139: 70}, 150)
    p = Pool(rng, lens, kv_heads, hd, 64, typ).fill()
    p.check(p.attend(new, heads, max_q=1200, pad=3), new)
