"""wv_decoder_forward_paged beyond single steps: what waits beside the running sequences, table widths, buffers that
stay over many calls, attention cut into key ranges and on tiles inside the decoder."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from test_gpu_serving import Server, config
from welvet_amd.kv import KVBatch

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


def test_buffers_stay():
    """A prompt of many rows and a chunk of fewer that needs more scratch (its attention's key ranges), in turn:
    neither frees what the other made."""
    cfg = config(32, 8, 128, n_layers=1, max_seq=1024)
    s = Server(cfg, "Q4_K", "q8", 1, width=256)
    ids, free = np.random.default_rng(6).integers(0, cfg.vocab, 600), []
    for _ in range(3):
        for call in (lambda: s.dec.prefill(ids), lambda: s.dec.forward_paged(s.kv, [ids[:256]], [7936], s.pages)):
            call()
            torch.cuda.synchronize()
            free.append(torch.cuda.mem_get_info()[0])
    print("[gpu] free", [f >> 20 for f in free], flush=True)
    assert len(set(free[1:])) == 1, free


def test_buffers_grow_by_more_than_a_row():
    """A sequence more in every call: buffers are not made anew for each."""
    cfg = config(8, 2, 64, n_layers=1, hidden=512, ffn=131072)
    s = Server(cfg, "Q4_K", "q8", 96, width=1)
    free = []
    for n in range(40, 97):
        s.dec.forward_paged(s.kv, [[1]] * n, [0] * n, s.pages[:n])
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    print("[gpu] free", [f >> 20 for f in free], flush=True)
    # rows, scratch, operands and logits: each by half at least, so three times from 40 to 96
    assert len(set(free)) <= 13, free


def splits(s, new):
    """Whether attention over the longest sequence's pages is cut into key ranges for these new tokens."""
    longest = max(len(i) + n for i, n in zip(s.ids, new) if n)
    b = KVBatch(len(new), sum(new), -(-longest // s.page), 0, 0, 0, max_q=max(new))
    return s.kv.attention_scratch(b, s.cfg.n_heads) > 0


@pytest.mark.parametrize("typ", ["f16", "q8"])
def test_key_ranges(typ):
    """Tokens behind a prompt of some hundreds: ranges and their join, in the buffer of the projections' partials."""
    cfg = config(8, 2, 64, n_layers=2)
    s = Server(cfg, "Q4_K", typ, 2, width=32)
    rng = np.random.default_rng(3)
    s.step([rng.integers(0, cfg.vocab, 900), rng.integers(0, cfg.vocab, 20)])
    for lens in ((1, 1), (2, 0)):
        new = [rng.integers(0, cfg.vocab, n) for n in lens]
        assert splits(s, lens)
        tokens, logits = s.step(new)
        s.check(new, tokens, logits, 2e-3)


@pytest.mark.parametrize("typ", ["f16", "q8"])
def test_tiles(typ):
    """A prompt that the tile kernel takes beside a short one."""
    cfg = config(32, 8, 128, n_layers=1)
    s = Server(cfg, "Q4_K", typ, 2, width=52)
    rng = np.random.default_rng(4)
    new = [rng.integers(0, cfg.vocab, n) for n in (1600, 3)]
    tokens, logits = s.step(new)
    s.check(new, tokens, logits, 2e-3)
