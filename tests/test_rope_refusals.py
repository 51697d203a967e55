"""Refusals of rotary positions that need no device."""
import math

import pytest

import welvet_amd as wv
from welvet_amd.rope import Rope

OK = dict(head_dim=64, theta=1e4)
RAMP = dict(scaling="ramp_dims", factor=4.0, trained=2048, low=1.0, high=32.0)


@pytest.mark.parametrize("bad,code,text", [
    (dict(head_dim=0), -2, "values of a head"), (dict(head_dim=1026), -2, "values of a head"),
    (dict(rot_dim=0), -2, "values of a head"), (dict(rot_dim=66), -2, "values of a head"),
    (dict(rot_dim=31), -2, "values of a head"), (dict(rot_dim=-2), -2, "values of a head"),
    (dict(layout=2), -1, "layout 2"), (dict(scaling=5), -1, "scaling 5"), (dict(scaling=-1), -1, "scaling -1"),
    (dict(theta=1.0), -1, "theta"), (dict(theta=math.nan), -1, "theta"), (dict(theta=math.inf), -1, "theta"),
    (dict(gain=0.0), -1, "gain"), (dict(gain=-1.0), -1, "gain"), (dict(gain=math.inf), -1, "gain"),
    (dict(scaling="linear", factor=0.0), -1, "factor"), (dict(scaling="linear", factor=math.nan), -1, "factor"),
    (dict(scaling="base", factor=2.0, rot_dim=2), -1, "factor"), (dict(scaling="base", factor=1e-9), -1, "factor"),
    (RAMP | dict(trained=0), -1, "trained"), (RAMP | dict(low=0.0), -1, "turns"), (RAMP | dict(high=1.0), -1, "turns"),
    (RAMP | dict(high=math.inf), -1, "turns"), (RAMP | dict(scaling="ramp_turns", low=40.0), -1, "turns"),
])
def test_create_refusals(bad, code, text):
    with pytest.raises(wv.WelvetError) as e:
        Rope(**(OK | bad))
    assert e.value.code == code and text in str(e.value)


def test_nil_and_unknown():
    L = wv.lib()
    assert L.wv_rope_create(None, None) == -1
    assert L.wv_rope_free(987654) == -7
    assert L.wv_rope_dev(987654, None, 1, None, None, None) == -7
    assert b"unknown rope" in L.wv_last_error()
