"""Settings whose numbers leave their type: refused before a device is asked for."""
import pytest

import welvet_amd as wv
from welvet_amd.rope import Rope

RAMP = dict(trained=64, low=1.0, high=4.0)


@pytest.mark.parametrize("bad,text", [
    (dict(scaling="linear", factor=1e-320), "frequencies"), (dict(scaling="linear", factor=5e-324), "frequencies"),
    (dict(scaling="ramp_dims", factor=1e-320, **RAMP), "frequencies"),
    (dict(scaling="ramp_turns", factor=1e-320, **RAMP), "frequencies"),
    (dict(gain=1e39), "gain"), (dict(gain=1e-46), "gain"),
])
def test_out_of_range(bad, text):
    with pytest.raises(wv.WelvetError) as e:
        Rope(64, theta=1e4, **bad)
    assert e.value.code == -1 and text in str(e.value)
