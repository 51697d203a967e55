"""The operators of a serving step, as cases that can be timed: the paged KV
cache that several sequences share (written in fp16 or int8 codes with a scale
per token and KV head, and read back), the attention of new tokens over it,
and the draw of each sequence's next token.

A case is one pass through one of them. Head layouts and widths are those of
bench.py's decoder and of the tests (32 query heads over 8 KV heads of 128,
heads of 64; vocabulary 32000), lengths go from one token to a cache of 131071
positions, ragged batches among them.

Definitions (what both forms of run() compute):
  cache row  x of one token and KV head, amax = max |x|:
             f16: s = 2^(floor(log2 amax) - 14), code = f16(x / s)
             q8:  s = f32(amax / 127), code = x / s rounded half away from zero
             read back: code * s
  attention  query i of a sequence with n new tokens and kv_len keys stands at
             position kv_len - n + i and attends keys j <= its position (and
             j > position - window, with a window)
  sample     w = exp((logit - max) / T); tokens in order of falling logit, equal
             ones by index; the first top_k of them; the shortest prefix of
             those that holds top_p of their mass; of these w >= min_p; the
             token is the first by index at which the running sum of w passes
             u times its total. T <= 0: the largest logit's first index.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # The draw of one sequence's next token at the decoder's vocabulary: latency.
        dict(name="sample_one", kind="sample", rows=1, vocab=32000, pad=0, filters="kp"),
        # A batch at a large vocabulary, nucleus and min-p: every logit of every row counts.
        dict(name="sample_nucleus", kind="sample", rows=64, vocab=128000, pad=0, filters="pm"),
        # A large serving batch whose requests each bring their own settings, greedy ones among them; rows padded.
        dict(name="sample_mixed", kind="sample", rows=256, vocab=32000, pad=5, filters="mixed"),
        # A decode step's new rows: one token of each of 64 sequences.
        dict(name="cache_tokens", kind="cache", type="q8", kv_heads=8, hd=128, page=32, rows=64, back=64),
        # A prompt's rows, the longest that a 2048-position cache takes, written and read back.
        dict(name="cache_prompt", kind="cache", type="f16", kv_heads=8, hd=128, page=32, rows=2047, back=2047),
        # A chunk appended to a long sequence, which is then read out whole (swapped to another device or program).
        dict(name="cache_bulk", kind="cache", type="q8", kv_heads=8, hd=128, page=64, rows=512, back=16384),
        # A decode step of one sequence at the bench's 2048 positions: the smallest attention call.
        dict(name="token_2k", kind="attn", type="q8", heads=32, kv_heads=8, hd=128, page=32, seqs=1, kv=2048, new=1,
             chunks=0, window=0),
        # A decode step of 64 sequences of ragged lengths: bytes of the cache.
        dict(name="tokens_64", kind="attn", type="q8", heads=32, kv_heads=8, hd=128, page=64, seqs=64, kv=8192, new=1,
             chunks=0, window=0),
        # One long context, one token: few rows over a long axis.
        dict(name="token_long", kind="attn", type="f16", heads=32, kv_heads=8, hd=128, page=128, seqs=1, kv=131071,
             new=1, chunks=0, window=0),
        # A whole prompt in one chunk.
        dict(name="prompt_2k", kind="attn", type="f16", heads=32, kv_heads=8, hd=128, page=32, seqs=1, kv=2047,
             new=2047, chunks=1, window=0),
        # A chunk of a long prompt over what earlier chunks left in the cache: the largest call.
        dict(name="chunk_16k", kind="attn", type="q8", heads=32, kv_heads=8, hd=128, page=64, seqs=1, kv=16384,
             new=2048, chunks=1, window=0),
        # A mixed step: prompt chunks beside decoding sequences, one of them idle, a sliding window, heads of 64.
        dict(name="mixed_window", kind="attn", type="f16", heads=16, kv_heads=8, hd=64, page=32, seqs=24, kv=4096,
             new=256, chunks=4, window=1024),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("sample", "cache", "attn", "attn", "attn"))
    typ = rng.choice(("f16", "q8"))
    if kind == "sample":
        vocab = _log_int(rng, 1000, 131072)
        return dict(kind=kind, rows=_log_int(rng, 1, min(256, (64 * 128000) // vocab)), vocab=vocab,
                    pad=rng.choice((0, 0, 5)), filters=rng.choice(("", "k", "p", "m", "kp", "kpm", "mixed")))
    kv_heads, hd, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 128)), rng.choice((32, 64, 128))
    if kind == "cache":
        rows = _log_int(rng, 1, 4096)
        return dict(kind=kind, type=typ, kv_heads=kv_heads, hd=hd, page=page, rows=rows,
                    back=_log_int(rng, rows, 16384))
    group = rng.choice((1, 2, 3, 4) if kv_heads == 8 else (1, 2, 3, 4, 8))
    c = dict(kind=kind, type=typ, heads=kv_heads * group, kv_heads=kv_heads, hd=hd, page=page)
    window = rng.choice((0, 0, 0, 257, 1024))
    shape = rng.choice(("one", "tokens", "chunk", "mixed"))
    if shape == "one":  # one sequence, one or a few new tokens
        return c | dict(seqs=1, kv=_log_int(rng, 16, 131072), new=rng.choice((1, 1, 2, 5)), chunks=1, window=window)
    if shape == "tokens":
        seqs = _log_int(rng, 2, 128)
        return c | dict(seqs=seqs, kv=_log_int(rng, 16, min(16384, 524288 // seqs)), new=1, chunks=0, window=window)
    if shape == "chunk":
        new = _log_int(rng, 16, 2048)
        return c | dict(seqs=1, kv=_log_int(rng, new, 16384), new=new, chunks=1, window=window)
    seqs = _log_int(rng, 2, 32)
    return c | dict(seqs=seqs, kv=_log_int(rng, 256, 4096), new=_log_int(rng, 2, 256), chunks=rng.randint(1, seqs),
                    window=window)


def _lengths(c):
    """(new tokens, keys) of each sequence: ragged, the same for every seed."""
    n, total = [], []
    r = random.Random(c["seqs"] * 1000003 + c["kv"] * 31 + c["new"])
    for i in range(c["seqs"]):
        new = c["new"] if c["seqs"] == 1 else r.randint(1, c["new"]) if i < c["chunks"] else 1
        if c["chunks"] and c["seqs"] > 4 and i == c["seqs"] - 2:
            new = 0  # idle in this step
        n.append(new)
        total.append(c["kv"] if c["seqs"] == 1 else max(new, r.randint(c["kv"] // 4, c["kv"])))
    return n, total


def _pairs(c):
    """(query, key) pairs that the mask leaves, and the keys that any query of their sequence sees."""
    pairs = keys = 0
    for n, total in zip(*_lengths(c)):
        first = total - n
        w = c["window"] or total + 1
        pairs += sum(min(p + 1, w) for p in range(first, total))
        keys += total - max(0, first - w + 1) if n else 0
    return pairs, keys


def _row_bytes(c):
    return c["kv_heads"] * (c["hd"] * (2 if c["type"] == "f16" else 1) + 4)


def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + c["rows"] * (5 * 4 + 8), "flops": 4 * n}
    if c["kind"] == "cache":
        f32 = 2 * c["kv_heads"] * c["hd"] * 4
        return {"bytes": (c["rows"] + c["back"]) * (f32 + 2 * _row_bytes(c) + 8),
                "flops": 3 * 2 * c["rows"] * c["kv_heads"] * c["hd"]}
    pairs, keys = _pairs(c)
    rows = sum(_lengths(c)[0])
    return {"bytes": 2 * keys * _row_bytes(c) + 2 * rows * c["heads"] * c["hd"] * 4,
            "flops": 4 * pairs * c["heads"] * c["hd"]}


# --------------------------------------------------------------- the inputs

def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1009 + salt) % (1 << 62))


def _rows(seed, salt, n, heads, hd, outliers):
    """Rows as projections leave them: normal, and for keys a few channels that stand out."""
    x = torch.randn(n, heads, hd, generator=_gen(seed, salt), device="cuda")
    if outliers:
        x[:, :, torch.randperm(hd, generator=_gen(seed, salt + 50), device="cuda")[:4]] *= 6.0
    return x


def _settings(c, seed):
    """temperature, top_k, top_p, min_p and u of each row."""
    r, f = c["rows"], c["filters"]
    g = _gen(seed, 70)

    def pick(values, dtype):
        v = torch.tensor(values, device="cuda", dtype=dtype)
        return v[torch.randint(0, len(values), (r,), generator=g, device="cuda")].contiguous()

    u = torch.rand(r, generator=g, device="cuda")
    if f == "mixed":
        return (pick((0.0, 0.6, 0.8, 1.0, 1.3), torch.float32), pick((0, 1, 20, 50, 400), torch.int32),
                pick((0.5, 0.9, 0.95, 1.0), torch.float32), pick((0.0, 0.0, 0.05), torch.float32), u)
    one = torch.ones(r, device="cuda")
    return (one * 0.8, torch.full((r,), 40 if "k" in f else 0, device="cuda", dtype=torch.int32),
            one * (0.95 if "p" in f else 1.0), one * (0.02 if "m" in f else 0.0), u)


def _pages(c, seed, lens):
    """A page table: each sequence's pages lie anywhere in the pool. (table, pages in the pool)"""
    width = max(1, max(-(-n // c["page"]) for n in lens))
    pool = len(lens) * width + 3
    perm = torch.randperm(pool, generator=_gen(seed, 60), device="cuda").to(torch.int32)
    return perm[: len(lens) * width].view(len(lens), width).contiguous(), pool


_stream = None


def _the_stream():
    """The program's stream: every call of a pass goes there."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream


def prepare(case, seed):
    c = case
    s = {"case": c, "stream": _the_stream()}
    if c["kind"] == "sample":
        # a peaked head over a long tail, as a language model's logits
        l = torch.randn(c["rows"], c["vocab"] + c["pad"], generator=_gen(seed, 1), device="cuda") * 2.5
        s["logits"] = l[:, : c["vocab"]]
        s["set"] = _settings(c, seed)
        s["tokens"] = torch.zeros(c["rows"], dtype=torch.int32, device="cuda")
        s["probs"] = torch.zeros(c["rows"], device="cuda")
        torch.cuda.synchronize()
        return s
    if c["kind"] == "cache":
        n, total = c["rows"], c["back"]
        s["table"], s["pool"] = _pages(c, seed, [total])
        pos = torch.arange(total, device="cuda")
        slots = s["table"][0].long()[pos // c["page"]] * c["page"] + pos % c["page"]
        s["back_slots"], s["new_slots"] = slots.contiguous(), slots[total - n:].contiguous()
        s["k"], s["v"] = (_rows(seed, i, n, c["kv_heads"], c["hd"], i == 1) for i in (1, 2))
        old = [_rows(seed, i, total - n, c["kv_heads"], c["hd"], i == 3) for i in (3, 4)]
        old_slots = slots[: total - n].contiguous()
        s["k_back"], s["v_back"] = (torch.zeros(total, c["kv_heads"], c["hd"], device="cuda") for _ in range(2))
    else:
        new, total = _lengths(c)
        s["new"], s["total"] = new, total
        s["table"], s["pool"] = _pages(c, seed, total)
        s["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        s["kv_len"] = torch.tensor(total, dtype=torch.int32, device="cuda")
        s["q"] = _rows(seed, 5, sum(new), c["heads"], c["hd"], False)
        s["out"] = torch.zeros_like(s["q"])
        width = s["table"].shape[1] * c["page"]
        pos = torch.arange(width, device="cuda")
        slots = s["table"].long()[:, pos // c["page"]] * c["page"] + pos % c["page"]
        old_slots = slots[pos[None, :] < s["kv_len"][:, None]]
        old = [_rows(seed, i, sum(total), c["kv_heads"], c["hd"], i == 3) for i in (3, 4)]
    if own:
        import welvet_amd as wv
        from welvet_amd.kv import KVBatch, KVCache
        wv.init(0)
        s["kv"] = KVCache(1, c["kv_heads"], c["hd"], c["page"], s["pool"], c["type"])
        torch.cuda.synchronize()
        s["kv"].write_dev(0, old[0].data_ptr(), old[1].data_ptr(), old_slots.data_ptr(), old_slots.numel(),
                          stream=s["stream"].cuda_stream)
        if c["kind"] == "attn":
            s["batch"] = KVBatch(c["seqs"], sum(s["new"]), s["table"].shape[1], s["cu"].data_ptr(),
                                 s["kv_len"].data_ptr(), s["table"].data_ptr(), max_q=max(s["new"]))
    else:
        s["cache"] = []
        for x in old:
            code, scale = _encode(x, c["type"])
            pool = s["pool"] * c["page"]
            codes = torch.zeros(pool, c["kv_heads"], c["hd"], dtype=code.dtype, device="cuda")
            scales = torch.zeros(pool, c["kv_heads"], 1, device="cuda")
            codes[old_slots], scales[old_slots] = code, scale
            s["cache"] += [codes, scales]
    torch.cuda.synchronize()
    return s


# ----------------------------------------------------------- the plain forms

def _encode(x, typ):
    """Codes and scales of rows, in 32 bits; the quotients next to a rounding border in 64."""
    amax = x.abs().amax(-1, keepdim=True)
    if typ == "f16":
        scale = torch.ldexp(torch.ones_like(amax), torch.frexp(amax).exponent - 15)
        return (x / scale).half(), scale
    scale = (amax.double() / 127.0).float()
    t = x.double() / scale.double()
    return (torch.sign(t) * torch.floor(t.abs() + 0.5)).clamp(-127, 127).to(torch.int8), scale


def _plain_cache(s):
    c = s["case"]
    for i, x in enumerate((s["k"], s["v"])):
        code, scale = _encode(x, c["type"])
        s["cache"][2 * i][s["new_slots"]] = code
        s["cache"][2 * i + 1][s["new_slots"]] = scale
    back = s["back_slots"]
    return tuple(s["cache"][2 * i][back].float() * s["cache"][2 * i + 1][back] for i in range(2))


def _plain_attention(s):
    c = s["case"]
    b, h, g, hd = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["hd"]
    nq, part = max(s["new"]), 512  # the sum over the keys in parts: a long one loses digits in 32 bits
    nk = -(-max(s["total"]) // part) * part
    dev = s["q"].device
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    i, j = torch.arange(nq, device=dev), torch.arange(nk, device=dev)
    rows = (s["cu"][:-1].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)  # [b, nq], padded
    page = (j // c["page"]).clamp(max=s["table"].shape[1] - 1)
    slots = s["table"].long()[:, page] * c["page"] + j % c["page"]  # [b, nk]
    k, v = ((s["cache"][2 * t][slots].float() * s["cache"][2 * t + 1][slots]).transpose(1, 2) for t in range(2))
    q = s["q"][rows].view(b, nq, h, g, hd).permute(0, 2, 3, 1, 4).reshape(b, h, g * nq, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(b, h, g, nq, nk) * (1.0 / math.sqrt(hd))
    pos = (s["kv_len"].long() - n)[:, None] + i  # [b, nq]
    seen = (j <= pos[:, :, None]) & (j < s["kv_len"].long()[:, None, None])
    if c["window"]:
        seen &= j > pos[:, :, None] - c["window"]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p = p.view(b, h, g * nq, nk // part, part).transpose(2, 3).contiguous()
    o = torch.matmul(p, v.reshape(b, h, nk // part, part, hd)).sum(2).view(b, h, g, nq, hd)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, nq, c["heads"], hd)
    return o[i[None, :] < n[:, None]]


def _plain_sample(s):
    l = s["logits"]
    t, top_k, top_p, min_p, u = (x[:, None] for x in s["set"])
    v = l.shape[1]
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    lmax = l.amax(1, keepdim=True).double()
    t = t.double()
    w = torch.exp((l.double() - lmax) / torch.where(t > 0, t, torch.ones_like(t)))  # sums next to a border: 64 bits
    rank = torch.arange(v, device=l.device)
    k = torch.where(top_k > 0, top_k, v).clamp(max=v)
    k = torch.where(t > 0, k, torch.ones_like(k))
    ws = torch.gather(w, 1, order) * (rank < k)
    before = torch.cumsum(ws, 1) - ws
    keep = (rank < k) & ((before < top_p.double() * ws.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0))
    keep &= ws >= min_p.double()
    w = torch.zeros_like(w).scatter_(1, order, ws * keep)
    run_sum = torch.cumsum(w, 1)
    total = run_sum[:, -1:]
    token = (run_sum <= u.double() * total).sum(1, keepdim=True).clamp(max=v - 1)
    prob = torch.gather(w, 1, token) / total
    return token[:, 0].to(torch.int32), prob[:, 0].float()


# ----------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    if not own:
        if c["kind"] == "sample":
            return dict(zip(("tokens", "probs"), _plain_sample(s)))
        if c["kind"] == "cache":
            return dict(zip(("k", "v"), _plain_cache(s)))
        return {"out": _plain_attention(s)}
    sh = s["stream"].cuda_stream
    if c["kind"] == "sample":
        from welvet_amd.sampling import sample_dev
        t, k, p, m, u = (x.data_ptr() for x in s["set"])
        sample_dev(s["logits"].data_ptr(), c["rows"], c["vocab"], s["tokens"].data_ptr(), u,
                   stride=s["logits"].stride(0), temperature_ptr=t, top_k_ptr=k, top_p_ptr=p, min_p_ptr=m,
                   probs_ptr=s["probs"].data_ptr(), stream=sh)
        return {"tokens": s["tokens"], "probs": s["probs"]}
    if c["kind"] == "cache":
        s["kv"].write_dev(0, s["k"].data_ptr(), s["v"].data_ptr(), s["new_slots"].data_ptr(), c["rows"], stream=sh)
        s["kv"].read_dev(0, s["back_slots"].data_ptr(), c["back"], s["k_back"].data_ptr(), s["v_back"].data_ptr(),
                         stream=sh)
        return {"k": s["k_back"], "v": s["v_back"]}
    s["kv"].attention_dev(0, s["batch"], s["q"].data_ptr(), s["out"].data_ptr(), c["heads"],
                          1.0 / math.sqrt(c["hd"]), window=c["window"], stream=sh)
    return {"out": s["out"]}


# ------------------------------------------------------ the exact results

def _stored(x, typ):
    """What the cache holds of rows x, in 64 bits."""
    y = x.double()
    top = y.abs().max(dim=-1, keepdim=True).values
    if typ == "f16":
        unit = torch.exp2(torch.floor(torch.log2(top)))
        unit = torch.where(unit > top, unit / 2, torch.where(2 * unit <= top, unit * 2, unit))  # log2 next to a power
        return (y / unit * 2.0 ** 14).to(torch.float16).double() * unit / 2.0 ** 14
    step = (top / 127).to(torch.float32).double()
    whole = torch.trunc(y / step)
    whole = whole + torch.where((y / step - whole).abs() >= 0.5, torch.sign(y), torch.zeros_like(y))
    return whole.clamp(-127, 127) * step


def _exact_attention(c, seed):
    new, total = _lengths(c)
    h, g, hd = c["kv_heads"], c["heads"] // c["kv_heads"], c["hd"]
    k = _stored(_rows(seed, 3, sum(total), h, hd, True), c["type"])
    v = _stored(_rows(seed, 4, sum(total), h, hd, False), c["type"])
    q = _rows(seed, 5, sum(new), c["heads"], hd, False).double()
    out = torch.zeros_like(q)
    q0 = k0 = 0
    for n, m in zip(new, total):
        pos = torch.arange(m - n, m, device="cuda")
        key = torch.arange(m, device="cuda")
        hide = key[None] > pos[:, None]
        if c["window"]:
            hide |= key[None] <= pos[:, None] - c["window"]
        for kh in range(h if n else 0):
            kk, vv = k[k0:k0 + m, kh], v[k0:k0 + m, kh]
            for qh in range(kh * g, kh * g + g):
                a = (q[q0:q0 + n, qh] @ kk.t().contiguous()) / math.sqrt(hd)
                a = torch.softmax(a.masked_fill(hide, -math.inf), dim=1)
                out[q0:q0 + n, qh] = a @ vv
        q0, k0 = q0 + n, k0 + m
    return out


def _exact_sample(c, seed):
    l = torch.randn(c["rows"], c["vocab"] + c["pad"], generator=_gen(seed, 1), device="cuda") * 2.5
    l = l[:, : c["vocab"]].cpu().numpy().astype(np.float64)
    t, top_k, top_p, min_p, u = (x.cpu().numpy() for x in _settings(c, seed))
    tokens, probs = np.zeros(c["rows"], np.int32), np.zeros(c["rows"])
    for r in range(c["rows"]):
        if t[r] <= 0:
            tokens[r], probs[r] = int(np.argmax(l[r])), 1.0
            continue
        order = np.lexsort((np.arange(c["vocab"]), -l[r]))
        if top_k[r] > 0:
            order = order[: top_k[r]]
        w = np.exp((l[r][order] - l[r].max()) / np.float64(t[r]))
        if top_p[r] < 1:
            mass = np.cumsum(w)
            order = order[: 1 + int(np.searchsorted(mass, np.float64(top_p[r]) * mass[-1], side="left"))]
            w = w[: order.size]
        order, w = order[w >= np.float64(min_p[r])], w[w >= np.float64(min_p[r])]
        by = np.argsort(order)
        mass = np.cumsum(w[by])
        at = int(np.searchsorted(mass, np.float64(u[r]) * mass[-1], side="right"))
        tokens[r], probs[r] = order[by][at], w[by][at] / mass[-1]
    return tokens, probs


def exact(case, seed):
    c = case
    if c["kind"] == "sample":
        tokens, probs = _exact_sample(c, seed)
        return {"tokens": torch.from_numpy(tokens), "probs": torch.from_numpy(probs)}
    if c["kind"] == "cache":
        n, old = c["rows"], c["back"] - c["rows"]
        return {name: torch.cat([_stored(_rows(seed, b, old, c["kv_heads"], c["hd"], b == 3), c["type"]),
                                 _stored(_rows(seed, a, n, c["kv_heads"], c["hd"], a == 1), c["type"])])
                for name, a, b in (("k", 1, 3), ("v", 2, 4))}
    return {"out": _exact_attention(c, seed)}
