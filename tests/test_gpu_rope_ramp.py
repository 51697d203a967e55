"""The ramp between pairs whose upper end lies behind the last pair, as published: the correction range ends at
rot_dim - 1 at most."""
import math

import numpy as np
import pytest

import welvet_amd as wv
from test_gpu_rope import check, dev
from welvet_amd.rope import Rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def ramped(rot, theta, factor, trained, low, high):
    """Frequencies by the published steps: the pair at which a number of turns is made, the range held to 0 and
    rot - 1, the mask, the blend. The published steps hold only the range's end to rot - 1. Where its beginning lies
    behind that (all pairs make more than `high` turns, the last case below), they would divide by a negative width;
    here the beginning is held to rot - 1 too, as the header says, and no pair is scaled."""
    at = lambda n: rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = min(max(math.floor(at(high)), 0), rot - 1), min(math.ceil(at(low)), rot - 1)
    if first == last:
        last += 0.001
    ramp = np.clip((np.arange(rot // 2) - first) / (last - first), 0, 1)
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    return f / factor * ramp + f * (1 - ramp), math.ceil(at(low))


@pytest.mark.parametrize("rot,theta,trained,low,high,over", [
    (128, 1e4, 65536, 1.0, 32.0, True), (128, 1e4, 131072, 1.0, 32.0, True), (64, 1e4, 1 << 20, 1.0, 32.0, True),
    (20, 100.0, 4096, 1.0, 4.0, True), (128, 1e4, 1 << 24, 0.5, 8.0, True), (128, 1e4, 4096, 1.0, 32.0, False),
    (96, 5e5, 8192, 1.0, 32.0, False), (64, 10.0, 1 << 30, 1.0, 2.0, True),
])
def test_published_range(rot, theta, trained, low, high, over):
    f, last = ramped(rot, theta, 4.0, trained, low, high)
    assert (last > rot // 2 - 1) == over
    hd, n = 128, 40
    rng = np.random.default_rng(rot)
    x = rng.standard_normal((n, 3, hd)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, n).astype(np.int32)
    d, p = dev(x), dev(pos)
    Rope(hd, rot, theta=theta, scaling="ramp_dims", factor=4.0, trained=trained, low=low, high=high).apply_dev(
        p.data_ptr(), n, d.data_ptr(), 3)
    wv.sync()
    check(d.cpu().numpy(), x, pos, f, "half", rot, 1.0)
