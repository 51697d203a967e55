"""wv_decoder_forward_paged beyond single steps: what waits beside the running sequences, table widths, buffers that
stay over many calls, attention cut into key ranges and on tiles inside the decoder."""
import numpy as np
import pytest

import welvet_amd as wv
from test_gpu_serving import Server, config

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


@pytest.mark.parametrize("idle", [2048, 1 << 17, 1 << 20, 2 ** 31 - 1])
def test_idle_sequences_do_not_steer(idle):
    """A running sequence's bits are the same whatever waits beside it. Q8_0: rows on the f32 GEMVs keep them apart."""
    cfg = config(8, 2, 64)
    s = Server(cfg, "Q8_0", "f16", 2, width=64)
    s.step([np.random.default_rng(5).integers(0, cfg.vocab, 1900), []])
    n = len(s.ids[0])
    wide = np.full((2, 4096), -1, np.int32)
    wide[:, :64] = s.pages
    for table in (s.pages, wide):
        want = s.dec.forward_paged(s.kv, [[7], []], [n, 0], table, want_logits=True)[1]
        got = s.dec.forward_paged(s.kv, [[7], []], [n, idle], table, want_logits=True)[1]
        assert np.array_equal(got[0], want[0])


def test_table_of_2_31_positions():
    """Positions are 32-bit numbers: a table of more is refused, as wv_kv_attention_dev does."""
    s = Server(config(8, 2, 64), "Q4_K", "q8", 1, page=256, width=1)
    table = np.full((1, 1 << 23), -1, np.int32)
    table[0, 0] = s.pages[0, 0]
    with pytest.raises(wv.WelvetError) as e:
        s.dec.forward_paged(s.kv, [[1]], [0], table)
    assert e.value.code == -2 and "2^31" in str(e.value)
    s.dec.forward_paged(s.kv, [[1]], [0], table[:, :-1])
