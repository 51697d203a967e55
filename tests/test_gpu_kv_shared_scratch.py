"""Scratch of attention over shared prefixes, sized before the arrays are there."""
import pytest

import welvet_amd as wv
from welvet_amd.kv import KVBatch, KVCache, KVGroups

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


@pytest.mark.parametrize("seqs,tokens,pages,groups,shared", [(64, 64, 256, 1, 8192), (8, 8, 18, 1, 513), (1, 1, 4, 1, 0),
                                                             (70, 200, 2048, 3, 0), (5, 0, 4, 2, 0)])
def test_sizes_alone(seqs, tokens, pages, groups, shared):
    """The same bytes with and without arrays, which are not read."""
    kv = KVCache(1, 2, 64, 32, 4)
    with_arrays = kv.attention_shared_scratch(KVBatch(seqs, tokens, pages, 4096, 4096, 4096),
                                              KVGroups(groups, 4096, 4096, shared), 8)
    assert kv.attention_shared_scratch(KVBatch(seqs, tokens, pages, 0, 0, 0), KVGroups(groups, 0, 0, shared),
                                       8) == with_arrays
    assert with_arrays > 0 or seqs < 64
    for bad, text in ((KVGroups(-1, 0, 0), "-1 groups"), (KVGroups(1, 0, 0, -1), "max_shared -1"),
                      (KVGroups((1 << 24) + 1, 0, 0), "groups")):
        with pytest.raises(wv.WelvetError) as e:
            kv.attention_shared_scratch(KVBatch(seqs, tokens, pages, 0, 0, 0), bad, 8)
        assert e.value.code == -2 and text in str(e.value)
