"""Draws whose list of candidates is long (top-k above 128 together with top-p): rows cut over blocks, where tokens
of several slices meet in one list, up to the list's end and past it, and rows done whole."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from test_gpu_sample import check, draw, logits
from welvet_amd.sampling import sample_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


@pytest.mark.parametrize("v", [9000, 33000, 131072])
@pytest.mark.parametrize("k", [127, 128, 129, 400, 511, 512, 513])
@pytest.mark.parametrize("p,m", [(0.9, None), (0.9, 0.02), (0.999, None)])
def test_long_lists(v, k, p, m):
    rng = np.random.default_rng(v + k)
    check(logits(rng, 8, v), t=0.9, k=k, p=p, m=m, u=rng.random(8, np.float32))


@pytest.mark.parametrize("k", [400, 512])
def test_list_overflows(k):
    """More tokens in the cut's bin than a list takes (logits close together, or equal): the row is done whole."""
    rng = np.random.default_rng(k)
    x = logits(rng, 6, 50000, 0.02)
    x[3] = np.float32(-1.5)
    x[4] = np.where(np.arange(50000) % 83 == 5, np.float32(2.0), np.float32(-3.0))
    x[5, :40000] = -np.inf
    check(x, t=1.0, k=k, p=0.9, u=rng.random(6, np.float32))


def test_mixed_lists():
    """Rows of every path side by side: lists, overflowing ones, whole rows, greedy and masked ones."""
    rng = np.random.default_rng(5)
    r, v = 60, 40000
    x = logits(rng, r, v)
    x[::7] *= np.float32(0.01)
    x[11], x[12, 6:] = -np.inf, -np.inf
    check(x, t=rng.choice([0, 0.7, 1.2], r), k=rng.choice([0, 1, 128, 129, 400, 512, 513, 4000], r),
          p=rng.choice([0.5, 0.95, 1.0], r), m=rng.choice([0, 0.01], r), u=rng.random(r, np.float32))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two devices")
def test_on_another_device_than_the_current_one():
    """Rows on the stream's device while another is the library's current one: the scratch is that device's too."""
    rng = np.random.default_rng(6)
    x, u = logits(rng, 5, 50000), rng.random(5, np.float32)
    want = draw(x, p=np.full(5, 0.9), u=u)[0]
    wv.init(1)
    wv.init(0)
    with torch.cuda.device(1):
        l, uu, p = (torch.from_numpy(a).cuda() for a in (x, u, np.full(5, 0.9, np.float32)))
        tok, st = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
        torch.cuda.synchronize()
        sample_dev(l.data_ptr(), 5, 50000, tok.data_ptr(), uu.data_ptr(), top_p_ptr=p.data_ptr(), stream=st.cuda_stream)
        st.synchronize()
        assert tok.cpu().numpy().tolist() == want.tolist()
