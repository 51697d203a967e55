"""Calls whose outputs are each other's rows: refused, nothing is written."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from welvet_amd.adapters import AdapterBatch, Adapters, apply_dev
from welvet_amd.rope import Rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def test_adapters():
    """Two sets with one y, a y that is another's base or x; one handle twice with rows of its own is fine."""
    s = Adapters(64, 64, 4, 1, "f16")
    a, b = np.full((4, 64), 0.5, np.float16), np.full((64, 4), 0.25, np.float16)
    s.set(0, a, b, 1.0)
    x, y, z = (torch.full((3, 64), v, device="cuda") for v in (1.0, 2.0, 3.0))
    cu, ids = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1, 3], [0, 0]))
    torch.cuda.synchronize()
    px, py, pz = (t.data_ptr() for t in (x, y, z))
    batch = AdapterBatch(2, 3, cu.data_ptr(), ids.data_ptr())
    for text, ys, bases in (("set 0 are those of set 1", [py, py], None), ("set 0 are those of set 1", [py, py], [pz, pz]),
                            ("set 1 are those of set 0", [py, pz], [pz, px]), ("set 1 are x", [py, px], None),
                            ("set 0 are those of set 1", [py, pz], [py, py])):
        with pytest.raises(wv.WelvetError) as e:
            apply_dev([s, s], batch, px, ys, base_ptrs=bases)
        assert e.value.code == -1 and text in str(e.value)
    wv.sync()
    assert all((t == v).all() for t, v in ((x, 1.0), (y, 2.0), (z, 3.0)))
    apply_dev([s, s], batch, px, [py, pz])
    wv.sync()
    add = 64 * 0.5 * 4 * 0.25  # sums of whole numbers: exact
    assert (y == 2.0 + add).all() and (z == 3.0 + add).all()


def test_rope():
    """q and k that are the same rows, or one's output the other's input; one input for two outputs is fine."""
    r = Rope(8, theta=100.0)
    x, y, z = (torch.full((3, 2, 8), v, device="cuda") for v in (1.0, 2.0, 3.0))
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    p, px, py, pz = (t.data_ptr() for t in (pos, x, y, z))
    for kw in (dict(k_ptr=px), dict(k_ptr=py, k_out_ptr=px), dict(k_ptr=py, q_out_ptr=py),
               dict(k_ptr=px, q_out_ptr=pz, k_out_ptr=pz), dict(k_ptr=px, q_out_ptr=py)):
        with pytest.raises(wv.WelvetError) as e:
            r.apply_dev(p, 3, px, 2, n_kv_heads=2, **kw)
        assert e.value.code == -1 and "are those of k" in str(e.value)
    wv.sync()
    assert all((t == v).all() for t, v in ((x, 1.0), (y, 2.0), (z, 3.0)))
    r.apply_dev(p, 3, px, 2, px, 1, q_out_ptr=py, k_out_ptr=pz, k_stride=16, k_out_stride=16)
    wv.sync()
    assert (y == 1.0).all() and (z[:, 0] == 1.0).all() and (z[:, 1] == 3.0).all()
    r.apply_dev(p, 3, px, 2, px, 0)  # no heads of k
    wv.sync()
