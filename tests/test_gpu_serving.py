"""The decoder over a shared paged cache (wv_decoder_forward_paged) and with drawn tokens
(wv_decoder_generate_sampled): the cache's writes, the attention over it and the draw together, as a
server calls them step after step.

The reference is DecodeRef's arithmetic (oracle/decode_ref.py) with the K and V rows that the device's
cache holds, read back: what it makes of its own K and V rows may differ from those by the projections'
bar and one rounding of the cache's type (2^-11 of a value in fp16; 1 / 127 of the row's largest, a whole
step where the bar moves a quotient over its border, in int8). Logits then stand at the projections' bar:
2e-3 normwise on the fp16 GEMM (Q4_K, or more than 8 rows), 1e-5 on the f32 GEMVs (Q8_0 up to 8 rows)."""
import numpy as np
import pytest
import torch

import welvet_amd as wv
from oracle import decode_ref as dr
from test_gpu_prefill_decode import build, normwise
from test_gpu_sample import reference
from welvet_amd.decode import Config
from welvet_amd.kv import KVCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    print(f"[gpu] {__name__}: init device 0", flush=True)
    wv.init(0)
    yield


def config(heads=8, kv_heads=2, hd=64, **kw):
    return Config(**({"n_layers": 2, "hidden": 256, "n_heads": heads, "n_kv_heads": kv_heads, "head_dim": hd,
                      "ffn": 512, "vocab": 300, "max_seq": 64} | kw))


class Server:
    """Sequences over one cache, and their logits by the reference."""

    def __init__(self, cfg, fmt, typ, seqs, page=32, width=3, seed=1):
        self.cfg, self.typ = cfg, typ
        self.dec, self.ref = build(cfg, fmt, seed)
        rng = np.random.default_rng(seed)
        self.kv = KVCache(cfg.n_layers, cfg.n_kv_heads, cfg.head_dim, page, seqs * width + 1, typ)
        self.pages = rng.permutation(seqs * width + 1)[: seqs * width].reshape(seqs, width).astype(np.int32)
        self.page, self.ids = page, [[] for _ in range(seqs)]

    def step(self, new, **kw):
        out = self.dec.forward_paged(self.kv, new, [len(i) for i in self.ids], self.pages, want_logits=True, **kw)
        for i, n in zip(self.ids, new):
            i.extend(int(t) for t in n)
        return out

    def rows(self, layer, b):
        c, n = self.cfg, len(self.ids[b])
        j = np.arange(n)
        sl = torch.from_numpy(self.pages[b][j // self.page].astype(np.int64) * self.page + j % self.page).cuda()
        k, v = (torch.zeros(n, c.kv_dim, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        self.kv.read_dev(layer, sl.data_ptr(), n, k.data_ptr(), v.data_ptr())
        wv.sync()
        return k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64)

    def logits(self, b, bar):
        """The reference's logits after all ids of sequence b; checks the cache's rows on the way."""
        c, r, n = self.cfg, self.ref, len(self.ids[b])
        unit = 2.0 ** -11 if self.typ == "f16" else 1 / 127
        h = r.emb[np.clip(self.ids[b], 0, c.vocab - 1)].astype(np.float32)
        for L, (w, an, fn) in enumerate(r.layers):
            kd, vd = self.rows(L, b)
            for i in range(n):
                n1 = dr.rmsnorm(h[i], an, c.rms_eps)
                q, k, v = (w[x](n1).astype(np.float64) for x in "qkv")
                dr.rope(q, i, c.n_heads, c.head_dim, c.rope_theta)
                dr.rope(k, i, c.n_kv_heads, c.head_dim, c.rope_theta)
                for own, held in ((k, kd[i]), (v, vd[i])):
                    assert np.abs(own - held).max() <= (bar + unit) * np.abs(own).max() + 1e-30
                att = dr.attention(q, kd, vd, i + 1, c.n_heads, c.n_kv_heads, c.head_dim).astype(np.float32)
                x = (h[i] + w["o"](att)).astype(np.float32)
                n2 = dr.rmsnorm(x, fn, c.rms_eps)
                h[i] = x + w["down"](dr.silu_mul(w["gate"](n2), w["up"](n2)))
        return r.lm(dr.rmsnorm(h[n - 1], r.final_norm, c.rms_eps))

    def check(self, new, tokens, logits, bar):
        for b, n in enumerate(new):
            if not len(n):
                assert tokens[b] == -1 and not logits[b].any()
                continue
            ref = self.logits(b, bar)
            err = normwise(logits[b], ref)
            print(f"[gpu] sequence {b} after {len(self.ids[b])}: {err:.2e}", flush=True)
            assert err <= bar
            top = np.sort(ref)[-2:]
            if top[1] - top[0] > 2 * bar * np.abs(ref).max():
                assert tokens[b] == int(np.argmax(ref))


@pytest.mark.parametrize("typ", ["f16", "q8"])
@pytest.mark.parametrize("fmt,layout", [("Q4_K", (8, 2, 64)), ("Q8_0", (4, 1, 128)), ("Q6_K", (6, 2, 64)),
                                        ("Q4_K", (8, 8, 64))])
def test_sequences_step_by_step(typ, fmt, layout):
    """Prompts of several lengths, an idle sequence that joins later, chunks beside single tokens."""
    cfg = config(*layout)
    s = Server(cfg, fmt, typ, 3)
    rng = np.random.default_rng(4)
    draw = lambda n: rng.integers(0, cfg.vocab, n)  # noqa: E731
    for lens in ((33, 7, 0), (1, 1, 40), (1, 12, 1), (1, 1, 1)):
        new = [draw(n) for n in lens]
        tokens, logits = s.step(new)
        s.check(new, tokens, logits, 2e-3)


def test_few_rows_stand_at_the_f32_bar():
    """Q8_0 projections of up to 8 rows run on the f32 GEMVs, and attention adds no more than they do."""
    s = Server(config(4, 2, 64), "Q8_0", "f16", 2)
    for new in ([[1, 2, 3], [250, 7]], [[9], [11]], [[], [4, 5, 6, 7]]):
        tokens, logits = s.step(new)
        s.check(new, tokens, logits, 1e-5)


def test_drawn_tokens_follow_the_logits():
    cfg = config()
    s = Server(cfg, "Q4_K", "q8", 4)
    rng = np.random.default_rng(6)
    for lens in ((9, 20, 1, 0), (1, 1, 1, 5), (1, 0, 1, 1)):
        u = rng.random(4, np.float32)
        t, k = np.array([0.8, 0.0, 1.2, 1.0], np.float32), np.array([0, 5, 40, 300], np.int32)
        p, m = np.array([0.9, 1.0, 1.0, 0.5], np.float32), np.array([0, 0, 0.05, 0], np.float32)
        tokens, logits = s.step([rng.integers(0, cfg.vocab, n) for n in lens], uniform=u, temperature=t, top_k=k,
                                top_p=p, min_p=m)
        for b, n in enumerate(lens):
            assert (reference(logits[b], t[b], k[b], p[b], m[b], u[b])[2](int(tokens[b])) if n else tokens[b] == -1)


def test_shared_prefix_pages():
    """Two sequences over the same prompt pages, each going on in pages of its own."""
    cfg = config()
    s = Server(cfg, "Q4_K", "f16", 2)
    prompt = np.random.default_rng(8).integers(0, cfg.vocab, 32)
    s.step([prompt, []])
    s.pages[1, 0], s.ids[1] = s.pages[0, 0], list(s.ids[0])
    new = [[5], [6]]
    tokens, logits = s.step(new)
    s.check(new, tokens, logits, 2e-3)


def test_same_call_again_gives_the_same_bits():
    cfg = config(hidden=512)
    out = []
    for _ in range(2):
        s = Server(cfg, "Q4_K", "q8", 3)
        rng = np.random.default_rng(9)
        s.step([rng.integers(0, cfg.vocab, n) for n in (40, 3, 17)])
        out.append(s.step([[1], [2], [3]], uniform=[0.1, 0.5, 0.9], temperature=1.0))
    assert np.array_equal(out[0][0], out[1][0]) and np.array_equal(out[0][1], out[1][1])


def test_follows_the_librarys_stream():
    """Rows that calls without a stream still have to write when the forward is called are there for it."""
    cfg = config()
    s = Server(cfg, "Q4_K", "f16", 1)
    s.step([np.random.default_rng(3).integers(0, cfg.vocab, 60)])
    n = len(s.ids[0])
    j = np.arange(n)
    sl = torch.from_numpy(s.pages[0][j // s.page].astype(np.int64) * s.page + j % s.page).cuda()
    rows = [[torch.zeros(n, cfg.kv_dim, device="cuda") for _ in range(2)] for _ in range(cfg.n_layers)]
    zero, sink = torch.zeros(n, cfg.kv_dim, device="cuda"), torch.zeros(1 << 17, cfg.kv_dim, device="cuda")
    every = torch.zeros(1 << 17, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for L, (k, v) in enumerate(rows):
        s.kv.read_dev(L, sl.data_ptr(), n, k.data_ptr(), v.data_ptr())
    _, want = s.dec.forward_paged(s.kv, [[7]], [n], s.pages, want_logits=True)
    for L in range(cfg.n_layers):
        s.kv.write_dev(L, zero.data_ptr(), zero.data_ptr(), sl.data_ptr(), n)
    for _ in range(50):  # some milliseconds of other work in front of the rows
        s.kv.read_dev(0, every.data_ptr(), 1 << 17, sink.data_ptr(), sink.data_ptr())
    for L, (k, v) in enumerate(rows):
        s.kv.write_dev(L, k.data_ptr(), v.data_ptr(), sl.data_ptr(), n)
    _, got = s.dec.forward_paged(s.kv, [[7]], [n], s.pages, want_logits=True)
    assert np.array_equal(got, want)


def test_refusals():
    cfg = config()
    s = Server(cfg, "Q4_K", "q8", 2, width=1)
    d, kv, pg = s.dec, s.kv, s.pages

    def refused(code, text, fn, *a, **kw):
        with pytest.raises(wv.WelvetError) as e:
            fn(*a, **kw)
        assert e.value.code == code and text in str(e.value)

    refused(-1, "empty ids", d.forward_paged, kv, [[], []], [0, 0], pg)
    refused(-2, "exceed 32 positions", d.forward_paged, kv, [[1] * 3, []], [30, 0], pg)
    refused(-2, "after -1", d.forward_paged, kv, [[1], []], [-1, 0], pg)
    refused(-2, "page 3 of 3", d.forward_paged, kv, [[1], [2]], [0, 0], np.array([[0], [3]]))
    refused(-2, "page -1 of 3", d.forward_paged, kv, [[1], [2]], [0, 0], np.array([[-1], [0]]))
    refused(-2, "one position", d.forward_paged, kv, [[1], [2]], [4, 4], np.array([[0], [0]]))
    other = KVCache(1, cfg.n_kv_heads, cfg.head_dim, 32, 3, "q8")
    refused(-2, "cache of 1 layers", d.forward_paged, other, [[1], [2]], [0, 0], pg)
    other.handle, h = 987654321, other.handle
    refused(-7, "unknown cache", d.forward_paged, other, [[1], [2]], [0, 0], pg)
    other.handle = h
    d.forward_paged(kv, [[1], []], [31, 5], np.array([[pg[0, 0]], [99]]))  # an idle sequence's pages are not looked at
    refused(-2, "exceed max_seq", d.generate_sampled, 1, 60, [0.5] * 5)
    refused(-1, "step count", d.generate_sampled, 1, 0, [0.5] * 65)


def test_generate_sampled():
    """Steps one by one, in one call, and from a replayed graph draw the same tokens; each fits its logits."""
    cfg = config(vocab=1000)
    dec, ref = build(cfg, "Q4_K", 3)
    prompt = np.random.default_rng(5).integers(0, cfg.vocab, 20)
    u = np.random.default_rng(6).random(12, np.float32)
    kw = dict(temperature=0.9, top_k=200, top_p=0.95, min_p=0.001)
    first = dec.prefill(prompt)
    tok, one = first, []
    for i in range(12):
        t, logits = dec.generate_sampled(tok, 20 + i, u[i:i + 1], want_logits=True, **kw)
        assert reference(logits, *(np.float32(kw[x]) if x != "top_k" else kw[x]
                                   for x in ("temperature", "top_k", "top_p", "min_p")), u[i])[2](int(t[0]))
        tok = int(t[0])
        one.append(tok)
    assert len(set(one)) > 3
    for graph in (False, True, True):
        dec.use_graph(graph)
        dec.prefill(prompt)
        assert dec.generate_sampled(first, 20, u, **kw).tolist() == one
        dec.prefill(prompt)
        greedy = dec.generate(first, 20, 6).tolist()  # between them: the greedy step's own graph
        dec.prefill(prompt)
        assert dec.generate_sampled(first, 20, u[:6], temperature=0.0).tolist() == greedy
    assert dec.generate_sampled(first, 20, []).size == 0


def test_generate_sampled_large_vocab():
    """More logits than one block holds: the draw is cut over blocks, eager and in the replayed graph."""
    cfg = config(vocab=40000, n_layers=1)
    dec, _ = build(cfg, "Q4_K", 11)
    u = np.random.default_rng(12).random(6, np.float32)
    kw = dict(temperature=1.1, top_p=0.97, min_p=0.0001)
    tok, one = 5, []
    for i in range(6):
        t, logits = dec.generate_sampled(tok, i, u[i:i + 1], want_logits=True, **kw)
        assert reference(logits, np.float32(1.1), 0, np.float32(0.97), np.float32(0.0001), u[i])[2](int(t[0]))
        tok = int(t[0])
        one.append(tok)
    for graph in (False, True, True):
        dec.use_graph(graph)
        assert dec.generate_sampled(5, 0, u, **kw).tolist() == one
    s = Server(cfg, "Q4_K", "q8", 3, seed=11)
    tokens, logits = s.step([[1, 2], [], [7]], uniform=[0.3, 0.5, 0.8], temperature=1.1, top_k=900, top_p=0.9)
    for b, un in ((0, 0.3), (2, 0.8)):
        assert reference(logits[b], np.float32(1.1), 900, np.float32(0.9), 0, np.float32(un))[2](int(tokens[b]))
    assert tokens[1] == -1
