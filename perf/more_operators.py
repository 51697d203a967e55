"""Operators of a served batch of requests, as cases that can be timed: the
bookkeeping of a paged KV cache's pages (sequences forked, resized with copy on
write, the pool compacted), attention of a batch whose sequences share a long
prefix, rotary positions of query and key rows, and the requests' low-rank
adapters beside a shared projection.

A case is one pass through one of them. Widths are those of bench.py's decoder
and of the tests (hidden 4096, 14336 and 1024, 32 query heads over 8 KV heads of
128, heads of 64), lengths go from one token to 32768 shared positions.

Definitions (what both forms of run() compute), P(n) = ceil(n / page size):
  fork      table row b becomes row parent[b] as it was (parent -1: empty, b
            itself: unchanged); refs[p] counts the sequences that hold page p.
  resize    sequence b to length new[b]. First all that shrink give pages back.
            Then those that grow, by index: where the page that its next
            position lies in has rows of its own and is held by others too, it
            is copied to a free page; of sequences that grow from one page and
            are all its holders, the last keeps it. Then free pages for the
            rest; always the lowest free ones. From the first sequence on that
            does not find enough, growing ones stay as they are (ok 0).
  compact   with U pages held, the i-th held page from U on moves to the i-th
            free one below U.
  shared    causal attention of new tokens over their sequence's keys; the
            sequences of a group hold the same first `shared` positions.
  rope      (a, b) -> gain (a cos t - b sin t, a sin t + b cos t), t = position f_i,
            pair i of rot/2: (i, i + rot/2) or (2i, 2i + 1), the rest of a head
            as it is. f_i = theta^(-2i/rot); linear: f_i / factor; base: theta
            factor^(rot/(rot-2)); ramps: f_i (1 - r) / factor + f_i r, with
            n_i = trained f_i / 2 pi turns: r = (n_i - low) / (high - low) in
            [0, 1] (ramp_turns), or 1 - (i - i0) / (i1 - i0) in [0, 1], i0 and
            i1 the floor and the ceiling of the i with n_i = high and n_i = low,
            within 0 and rot/2 - 1, i1 at least 0.001 over i0 (ramp_dims).
  adapters  y_t = base_t + s_a B_a (A_a x_t), a the adapter of t's sequence.
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
        # A step of 8 beams that trade places: one layer group of a short sequence, latency.
        dict(name="fork_beams", kind="pages", op="fork", type="q8", layers=2, kv_heads=8, hd=128, page=32, groups=1,
             each=8, length=715, new=1, spare=9),
        # 16 prompts sampled 16 times each: forked, their last pages copied, room for the next tokens.
        dict(name="fork_samples", kind="pages", op="fork", type="f16", layers=4, kv_heads=8, hd=128, page=64, groups=16,
             each=16, length=4113, new=5, spare=40),
        # A pool after half of its sequences have ended: the others' pages move to its front.
        dict(name="compact_pool", kind="pages", op="compact", type="q8", layers=2, kv_heads=8, hd=128, page=64,
             groups=1, each=64, length=1500, new=0, spare=100),
        # One prompt answered 8 times: short, latency.
        dict(name="share_8", kind="shared", type="q8", heads=32, kv_heads=8, hd=128, page=32, groups=1, each=8, lone=0,
             shared=513, tail=64, new=1, window=0),
        # A batch of 64 requests behind one long instruction.
        dict(name="share_64", kind="shared", type="q8", heads=32, kv_heads=8, hd=128, page=64, groups=1, each=64,
             lone=0, shared=8192, tail=1024, new=1, window=0),
        # Questions of up to 100 tokens to a long document, read in one call.
        dict(name="share_questions", kind="shared", type="f16", heads=32, kv_heads=8, hd=128, page=32, groups=1,
             each=12, lone=0, shared=32768, tail=150, new=100, window=0),
        # Several groups of several sizes and sequences of no group, a few tokens to check for each, heads of 64.
        dict(name="share_groups", kind="shared", type="f16", heads=16, kv_heads=8, hd=64, page=32, groups=5, each=16,
             lone=7, shared=4096, tail=300, new=4, window=0),
        # One token's heads.
        dict(name="rope_token", kind="rope", heads=32, kv_heads=8, hd=128, rot=128, layout="half", scaling="none",
             rows=1, far=2048),
        # A prompt's rows far behind the trained length: pairs, half of the head.
        dict(name="rope_prompt", kind="rope", heads=32, kv_heads=8, hd=128, rot=64, layout="pairs", scaling="ramp_dims",
             rows=8191, far=131072),
        # One token of one request at a wide projection: latency.
        dict(name="adapt_token", kind="adapters", type="f16", rows=14336, sets=2, cols=4096, rank=16, adapters=4,
             seqs=1, new=1, chunks=0),
        # A decode step of 64 requests with 24 adapters between them at Q, K and V.
        dict(name="adapt_step", kind="adapters", type="bf16", rows=1024, sets=3, cols=4096, rank=32, adapters=24,
             seqs=64, new=1, chunks=0),
        # Prompts of several requests, and single tokens of others.
        dict(name="adapt_prompts", kind="adapters", type="bf16", rows=14336, sets=1, cols=4096, rank=64, adapters=6,
             seqs=12, new=700, chunks=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("pages", "shared", "shared", "rope", "adapters", "adapters"))
    typ = rng.choice(("f16", "q8"))
    if kind == "rope":
        hd = rng.choice((64, 80, 128, 256))
        kv_heads = rng.choice((1, 2, 4, 8))
        return dict(kind=kind, heads=kv_heads * rng.choice((1, 2, 4, 7)), kv_heads=kv_heads, hd=hd,
                    rot=rng.choice((hd, hd, hd // 2, 20)), layout=rng.choice(("half", "pairs")),
                    scaling=rng.choice(("none", "linear", "base", "ramp_dims", "ramp_turns")),
                    rows=_log_int(rng, 1, 8191), far=_log_int(rng, 100, 1 << 20))
    if kind == "adapters":
        c = dict(kind=kind, type=rng.choice(("f16", "bf16")), rows=_log_int(rng, 60, 14336), sets=rng.choice((1, 2, 3)),
                 cols=_log_int(rng, 60, 14336), rank=rng.choice((1, 4, 8, 16, 20, 32, 64, 128)))
        if rng.random() < 0.5:
            return c | dict(seqs=_log_int(rng, 1, 256), new=1, chunks=0,
                            adapters=_log_int(rng, 1, 32 if c["rank"] <= 32 else 8))
        seqs = _log_int(rng, 1, 16)
        return c | dict(seqs=seqs, new=_log_int(rng, 2, 300), chunks=rng.randint(1, min(seqs, 4)),
                        adapters=_log_int(rng, 1, 8))
    kv_heads, hd, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 128)), rng.choice((32, 64, 128))
    c = dict(kind=kind, type=typ, kv_heads=kv_heads, hd=hd, page=page)
    if kind == "pages":
        groups = _log_int(rng, 1, 16)
        each = _log_int(rng, 1, 16)
        return c | dict(op=rng.choice(("fork", "fork", "compact")), layers=rng.choice((1, 2, 4)), groups=groups,
                        each=each, length=_log_int(rng, 1, 4096), new=rng.choice((0, 1, 1, 5, 130)),
                        spare=rng.choice((0, 3, 100)))
    groups, each = _log_int(rng, 1, 6), _log_int(rng, 1, 64)
    seqs = groups * each
    c |= dict(heads=kv_heads * rng.choice((1, 2, 4) if kv_heads == 8 else (1, 3, 4, 8)), groups=groups, each=each,
              lone=rng.choice((0, 0, 1, 3)), window=rng.choice((0, 0, 0, 700)))
    c |= dict(shared=_log_int(rng, 16, min(32768, 390000 // seqs)), tail=_log_int(rng, 8, 1024))
    return c | dict(new=rng.choice((1, 1, 1, 3, 30)) if seqs > 16 else _log_int(rng, 1, 100))


def _rand(c):
    """The case's own random numbers: layouts that are the same for every seed."""
    return random.Random(sum(ord(ch) * 131 ** (i % 5) for i, ch in enumerate(repr(sorted(
        (k, v) for k, v in c.items() if k != "name")))))


# ------------------------------------------------- the layout of each case

def _share_plan(c):
    """Members of each group, shared positions, and (new tokens, keys) of each sequence; lone ones come last."""
    r = _rand(c)
    members = [c["each"]] if c["groups"] == 1 else [r.randint(1, c["each"]) for _ in range(c["groups"])]
    shared = [c["shared"] if g == 0 else r.randint(c["shared"] // 4, c["shared"]) for g in range(c["groups"])]
    new, total = [], []
    for g, m in enumerate(members + [1] * c["lone"]):
        for _ in range(m):
            n = c["new"] if not new else r.randint(1, c["new"])
            lead = shared[g] if g < c["groups"] else r.randint(0, c["shared"])
            new.append(n)
            total.append(lead + n + r.randint(0, max(0, c["tail"] - n)))
    return members, shared, new, total


def _share_tables(c, seed):
    """Page table (pages anywhere in the pool; a group's sequences hold the same pages of the prefix, as far as they
    are full), pool size, and the rows that fill the pool: (slots, sequence, position) of each, numpy."""
    members, shared, _, total = _share_plan(c)
    width = max(-(-n // c["page"]) for n in total)
    lead = np.zeros((len(total), 2), np.int64)  # first sequence of the group, shared full pages
    b = 0
    for g, m in enumerate(members):
        lead[b:b + m] = b, shared[g] // c["page"]
        b += m
    lead[b:, 0] = np.arange(b, len(total))
    held = [-(-n // c["page"]) for n in total]
    fresh = [n - int(lead[i, 1]) if lead[i, 0] != i else n for i, n in enumerate(held)]
    pool = sum(fresh) + 3
    perm = np.random.RandomState(seed % (1 << 31)).permutation(pool).astype(np.int32)
    table = np.full((len(total), width), -1, np.int32)
    slots, seq, pos = [], [], []
    at = 0
    for i, n in enumerate(held):
        f, k = int(lead[i, 0]), n - fresh[i]
        table[i, :k] = table[f, :k]
        table[i, k:n] = perm[at:at + fresh[i]]
        at += fresh[i]
        p = np.arange(k * c["page"], total[i])
        slots.append(table[i, p // c["page"]].astype(np.int64) * c["page"] + p % c["page"])
        seq.append(np.full(p.size, i))
        pos.append(p)
    return table, pool, np.concatenate(slots), np.concatenate(seq), np.concatenate(pos)


def _share_rows(c, seed, salt, outliers):
    """Rows of every sequence's keys, one after the other: [sum of keys, heads, hd], and where each sequence begins.
    A group's first rows are its first sequence's."""
    members, shared, _, total = _share_plan(c)
    start = np.concatenate([[0], np.cumsum(total)])
    x = _rows(seed, salt, int(start[-1]), c["kv_heads"], c["hd"], outliers)
    b = 0
    for g, m in enumerate(members):
        for i in range(b + 1, b + m):
            x[start[i]:start[i] + shared[g]] = x[start[b]:start[b] + shared[g]]
        b += m
    return x, start


def _adapt_plan(c):
    """Tokens and adapter of each sequence (-1: none), rank of each adapter."""
    r = _rand(c)
    new = [c["new"] if i == 0 and c["chunks"] else r.randint(1, c["new"]) if i < c["chunks"] else 1
           for i in range(c["seqs"])]
    which = [-1 if c["seqs"] > 3 and r.random() < 0.1 else r.randrange(c["adapters"]) for _ in range(c["seqs"])]
    which[0] = 0
    ranks = [c["rank"] if i == 0 else max(1, c["rank"] // r.choice((1, 1, 2))) for i in range(c["adapters"])]
    return new, which, ranks


def _adapt_rows(c):
    """Output rows of each set: the sets of one call need not be alike."""
    return [c["rows"] * 4 if c["sets"] == 3 and i == 0 and c["rows"] <= 2048 else c["rows"] for i in range(c["sets"])]


def _page_plan(c):
    """Start of a page case: lengths, table rows as lists, refs. Sequences hold whole pages of their own, one after
    the other, in a pool with `spare` pages left over; every group's first sequence is the one that is forked."""
    r = _rand(c)
    s = c["groups"] * c["each"]
    n = [max(1, c["length"] if i == 0 else r.randint(c["length"] // 2 + 1, c["length"])) for i in range(s)]
    held = [-(-x // c["page"]) for x in n]
    width = max(-(-(x + c["new"]) // c["page"]) for x in n) + 1
    return r, n, held, width


def _moves(c):
    """For work(): positions copied by a fork case (copies of last pages) and pages moved by a compact case."""
    _, n, held, _ = _page_plan(c)
    if c["op"] == "fork":
        off = [n[g * c["each"]] % c["page"] for g in range(c["groups"])]
        return sum(o * (c["each"] - 1) for o in off) if c["new"] else 0
    keep = [i for i in range(len(held)) if i % 2 or len(held) == 1]
    used = sum(held[i] for i in keep)
    first = np.concatenate([[0], np.cumsum(held)])
    return sum(int(np.sum(np.arange(first[i], first[i + 1]) >= used)) for i in keep)


def _row_bytes(c):
    return c["kv_heads"] * (c["hd"] * (2 if c["type"] == "f16" else 1) + 4)


def work(case):
    c = case
    if c["kind"] == "rope":
        n = c["rows"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 8 * n * c["hd"] + 4 * c["rows"], "flops": 3 * n * c["rot"]}
    if c["kind"] == "adapters":
        new, which, ranks = _adapt_plan(c)
        rows = _adapt_rows(c)
        used = {a for a in which if a >= 0}
        t = sum(new)
        w = sum(2 * ranks[a] * (c["cols"] + o) for a in used for o in rows)
        return {"bytes": w + 4 * t * c["cols"] + 8 * t * sum(rows),
                "flops": sum(2 * n * ranks[a] * (c["cols"] + o) for n, a in zip(new, which) if a >= 0 for o in rows)}
    if c["kind"] == "pages":
        _, n, held, width = _page_plan(c)
        moved = _moves(c) * (1 if c["op"] == "fork" else c["page"]) * c["layers"] * 2 * _row_bytes(c)
        back = sum(_back(c)) * c["layers"] * (2 * _row_bytes(c) + 8 * c["kv_heads"] * c["hd"])
        return {"bytes": 2 * moved + back + 8 * len(n) * width + 8 * sum(held), "flops": len(n) * width}
    members, shared, new, total = _share_plan(c)
    pairs = keys = b = 0
    for g, m in enumerate(members + [1] * c["lone"]):
        low, first = total[b], total[b]
        for i in range(b, b + m):
            w = c["window"] or total[i] + 1
            pos = total[i] - new[i]
            pairs += sum(min(p + 1, w) for p in range(pos, total[i]))
            first = max(0, pos - w + 1)
            lead = shared[g] if g < len(members) else 0
            keys += total[i] - max(first, lead)
            low = min(low, first)
        if g < len(members):
            keys += max(0, shared[g] - low)
        b += m
    return {"bytes": 2 * keys * _row_bytes(c) + 8 * sum(new) * c["heads"] * c["hd"],
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


def _ints(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dtype)


_stream = None


def _the_stream():
    """The program's stream: every call of a pass goes there."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream


def _back(c):
    """Rows of each sequence that a page case reads back: those of its last page before it grew, or all of them."""
    _, n, _, _ = _page_plan(c)
    if c["op"] == "fork":
        n = [n[i // c["each"] * c["each"]] for i in range(len(n))]
        return [x % c["page"] or c["page"] for x in n] if c["new"] else [min(x, c["page"]) for x in n]
    return [x if i % 2 or len(n) == 1 else 0 for i, x in enumerate(n)]


def _prepare_pages(s, c, seed):
    r, n, held, width = _page_plan(c)
    seqs, page = len(n), c["page"]
    lead = np.arange(seqs) // c["each"] * c["each"]
    parent = np.array([r.randrange(lead[i], lead[i] + c["each"]) if c["op"] == "fork" and c["new"] > 1 else lead[i]
                       for i in range(seqs)])
    if c["op"] == "fork":  # all sequences of a group as long as its first
        n = [n[lead[i]] for i in range(seqs)]
        held = [-(-x // page) for x in n]
    first = np.concatenate([[0], np.cumsum(held)])
    s["pool"] = int(first[-1]) + c["spare"] + (seqs * (width - min(held)) if c["op"] == "fork" else 0)
    table = np.full((seqs, width), -1, np.int32)
    refs = np.zeros(s["pool"], np.int32)
    for i in range(seqs):
        table[i, :held[i]] = np.arange(first[i], first[i + 1])
        refs[first[i]:first[i + 1]] = 1
    now = np.array(n)
    if c["op"] == "compact":  # every second sequence has ended
        for i in range(0, seqs if seqs > 1 else 0, 2):
            refs[first[i]:first[i + 1]] = 0
            table[i] = -1
            now[i] = 0
    packed = np.concatenate([table.reshape(-1), now, refs])
    s["start"] = _ints(packed)
    s["now"] = s["start"].clone()
    t, k = table.size, seqs
    s["table"], s["len"], s["refs"] = s["now"][:t].view(seqs, width), s["now"][t:t + k], s["now"][t + k:]
    s["parent"], s["base"], s["grown"] = _ints(parent), _ints(now), _ints(now + c["new"])
    s["ok"], s["used"] = _ints(np.zeros(seqs)), _ints(np.zeros(1))
    back = _back(c)
    s["back"] = back
    s["cu"] = _ints(np.concatenate([[0], np.cumsum(back)]))
    s["rows"] = sum(back)
    # the read-back's length of each sequence: its rows before it grew (fork), or all of it
    s["at"] = _ints(now)
    s["slots"] = torch.zeros(s["rows"], dtype=torch.int64, device="cuda")
    s["pos"] = torch.zeros(s["rows"], dtype=torch.int32, device="cuda")
    s["k"], s["v"] = (torch.zeros(c["layers"], s["rows"], c["kv_heads"], c["hd"], device="cuda") for _ in range(2))
    slots = np.concatenate([np.arange(first[i], first[i + 1])[np.arange(n[i]) // page] * page + np.arange(n[i]) % page
                            for i in range(seqs)])
    return _ints(slots, torch.int64), [[_rows(seed, 10 * l + i, len(slots), c["kv_heads"], c["hd"], i == 3)
                                        for i in (3, 4)] for l in range(c["layers"])]


def _rope_inputs(c, seed):
    g = _gen(seed, 5)
    q, k = (_rows(seed, i, c["rows"], h, c["hd"], False) for i, h in ((1, c["heads"]), (2, c["kv_heads"])))
    if c["rows"] > 256:  # a prompt's positions, ending at the last one
        pos = torch.arange(c["far"] - 1 - c["rows"], c["far"] - 1, device="cuda").clamp(min=0)
    else:
        pos = torch.randint(0, c["far"], (c["rows"],), generator=g, device="cuda")
    return q, k, pos.to(torch.int32)


#: theta, factor, trained positions, low and high turns, gain of a scaled rotation
_ROPE = dict(theta=5e5, factor=8.0, trained=8192, low=1.0, high=32.0, gain=1.1)


def _rope_settings(c):
    if c["scaling"] == "none":
        return dict(theta=_ROPE["theta"])
    if c["scaling"] in ("linear", "base"):
        return dict(theta=_ROPE["theta"], factor=_ROPE["factor"])
    return dict(_ROPE)


def _adapt_inputs(c, seed):
    new, which, ranks = _adapt_plan(c)
    dt = torch.float16 if c["type"] == "f16" else torch.bfloat16
    t = sum(new)
    x = torch.randn(t, c["cols"], generator=_gen(seed, 1), device="cuda")
    rows = _adapt_rows(c)
    base = [torch.randn(t, o, generator=_gen(seed, 20 + i), device="cuda") for i, o in enumerate(rows)]
    a, b = [], []
    for i, o in enumerate(rows):
        a.append([(torch.randn(r, c["cols"], generator=_gen(seed, 1000 + 100 * i + j), device="cuda")
                   / math.sqrt(c["cols"])).to(dt) for j, r in enumerate(ranks)])
        b.append([(torch.randn(o, r, generator=_gen(seed, 2000 + 100 * i + j), device="cuda") * 0.3).to(dt)
                  for j, r in enumerate(ranks)])
    scales = [2.0 if j % 2 == 0 else 0.75 for j in range(len(ranks))]
    return x, base, a, b, scales


def prepare(case, seed):
    c = case
    s = {"case": c, "stream": _the_stream()}
    if own:
        import welvet_amd as wv
        wv.init(0)
    sh = s["stream"].cuda_stream
    if c["kind"] == "rope":
        s["q"], s["k"], s["pos"] = _rope_inputs(c, seed)
        s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
        if own:
            from welvet_amd.rope import Rope
            s["rope"] = Rope(c["hd"], rot_dim=c["rot"], layout=c["layout"], scaling=c["scaling"], **_rope_settings(c))
        torch.cuda.synchronize()
        return s
    if c["kind"] == "adapters":
        new, which, ranks = _adapt_plan(c)
        s["x"], s["base"], a, b, scales = _adapt_inputs(c, seed)
        s["y"] = [torch.zeros_like(t) for t in s["base"]]
        s["cu"], s["which"] = _ints(np.concatenate([[0], np.cumsum(new)])), _ints(which)
        if own:
            from welvet_amd.adapters import AdapterBatch, Adapters
            s["sets"] = []
            for i, o in enumerate(_adapt_rows(c)):
                s["sets"].append(Adapters(o, c["cols"], max(ranks), len(ranks), c["type"]))
                for j in range(len(ranks)):
                    s["sets"][i].set(j, a[i][j].view(torch.int16).cpu().numpy().view(np.uint16),
                                     b[i][j].view(torch.int16).cpu().numpy().view(np.uint16), scales[j])
            s["batch"] = AdapterBatch(c["seqs"], sum(new), s["cu"].data_ptr(), s["which"].data_ptr(), max_q=max(new))
        else:
            r = max(ranks)
            s["a"] = [torch.nn.utils.rnn.pad_sequence(p, batch_first=True) for p in a]
            s["b"] = [torch.stack([torch.nn.functional.pad(t, (0, r - t.shape[1])) for t in p]) for p in b]
            s["scales"] = torch.tensor(scales, device="cuda")
            s["new"] = new
        torch.cuda.synchronize()
        return s
    if c["kind"] == "pages":
        old_slots, old = _prepare_pages(s, c, seed)
        layers = c["layers"]
    else:
        members, shared, new, total = _share_plan(c)
        s["new"], s["total"] = new, total
        table, s["pool"], slots, seq, pos = _share_tables(c, seed)
        s["table"] = _ints(table)
        s["cu"], s["kv_len"] = _ints(np.concatenate([[0], np.cumsum(new)])), _ints(total)
        s["group_cu"], s["shared"] = _ints(np.concatenate([[0], np.cumsum(members)])), _ints(shared)
        s["q"] = _rows(seed, 5, sum(new), c["heads"], c["hd"], False)
        s["out"] = torch.zeros_like(s["q"])
        old_slots, old = _ints(slots, torch.int64), [[]]
        for i in (3, 4):
            x, start = _share_rows(c, seed, i, i == 3)
            old[0].append(x[_ints(start[seq] + pos, torch.int64)])
        layers = 1
    if own:
        from welvet_amd.kv import KVBatch, KVCache, KVGroups, KVTables
        s["kv"] = KVCache(layers, c["kv_heads"], c["hd"], c["page"], s["pool"], c["type"])
        torch.cuda.synchronize()
        for l in range(layers):
            s["kv"].write_dev(l, old[l][0].data_ptr(), old[l][1].data_ptr(), old_slots.data_ptr(), old_slots.numel(),
                              stream=sh)
        if c["kind"] == "shared":
            s["batch"] = KVBatch(len(s["new"]), sum(s["new"]), s["table"].shape[1], s["cu"].data_ptr(),
                                 s["kv_len"].data_ptr(), s["table"].data_ptr(), max_q=max(s["new"]))
            s["groups"] = KVGroups(c["groups"], s["group_cu"].data_ptr(), s["shared"].data_ptr(),
                                   max_shared=max(shared))
        else:
            seqs, width = s["table"].shape
            s["work"] = torch.zeros(s["kv"].tables_work(seqs, width), dtype=torch.uint8, device="cuda")
            s["tables"] = KVTables(seqs, width, s["table"].data_ptr(), s["len"].data_ptr(), s["refs"].data_ptr(),
                                   s["work"].data_ptr())
            s["batch"] = KVBatch(seqs, s["rows"], width, s["cu"].data_ptr(), s["at"].data_ptr(), s["table"].data_ptr())
    else:
        pool = s["pool"] * c["page"]
        s["cache"] = []
        for i in range(2):
            for l in range(layers):
                code, scale = _encode(old[l][i], c["type"])
                if l == 0:
                    codes = torch.zeros(layers, pool, c["kv_heads"], c["hd"], dtype=code.dtype, device="cuda")
                    scales = torch.zeros(layers, pool, c["kv_heads"], 1, device="cuda")
                codes[l][old_slots], scales[l][old_slots] = code, scale
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


def _held(table, length, page):
    """Which table entries the sequences hold."""
    return torch.arange(table.shape[1], device=table.device) < ((length.long() + page - 1) // page)[:, None]


def _plain_fork(table, length, refs, parent, page):
    old = _held(table, length, page)
    gone = parent < 0
    src = parent.long().clamp(min=0)
    row, n = table[src], torch.where(gone, torch.zeros_like(length), length[src])
    new = _held(table, n, page)
    row = torch.where(new, row, torch.full_like(row, -1))
    refs.index_add_(0, row[new].long(), torch.ones_like(row[new]))
    refs.index_add_(0, table[old].long(), -torch.ones_like(table[old]))
    table.copy_(row)
    length.copy_(n)


def _plain_resize(table, length, refs, to, ok, page, pools):
    """Copies last pages in every tensor of `pools` ([layers, positions, ...])."""
    dev = table.device
    at = torch.arange(table.shape[1], device=dev)
    drop = _held(table, length, page) & ~_held(table, to, page)
    refs.index_add_(0, table[drop].long(), -torch.ones_like(table[drop]))
    table[drop] = -1
    length.copy_(torch.minimum(length, to))
    have, want = (length.long() + page - 1) // page, (to.long() + page - 1) // page
    grow = to > length
    part = grow & (length % page != 0)
    idx = (have - 1).clamp(min=0)
    last = torch.gather(table, 1, idx[:, None])[:, 0].long().clamp(min=0)
    same = (last[:, None] == last[None]) & part[:, None] & part[None]
    row = torch.arange(len(to), device=dev)
    later = (same & (row[None] > row[:, None])).any(1)
    copy = part & (refs[last] > 1) & ~((same.sum(1) == refs[last]) & ~later)
    need = torch.where(grow, want - have + copy, torch.zeros_like(want))
    end = torch.cumsum(need, 0)
    free = torch.nonzero(refs == 0)[:, 0]
    done = ~grow | (end <= free.numel())
    copy, serve = copy & done, grow & done
    first = have - copy.long()
    fresh = serve[:, None] & (at >= first[:, None]) & (at < want[:, None])
    took = free[((end - need - first)[:, None] + at)[fresh]]
    src = last[copy]
    refs.index_add_(0, src, -torch.ones_like(src, dtype=refs.dtype))
    table[fresh] = took.to(table.dtype)
    refs[took] = 1
    dst = torch.gather(table, 1, idx[:, None])[:, 0].long()[copy]
    for x in pools:
        x = x.view(x.shape[0], -1, page, *x.shape[2:])
        x[:, dst] = x[:, src]
    length.copy_(torch.where(serve, to, length))
    ok.copy_(done)


def _plain_compact(table, length, refs, used, page, pools):
    held = refs > 0
    u = int(held.sum())
    holes, movers = torch.nonzero(~held[:u])[:, 0], torch.nonzero(held[u:])[:, 0] + u
    to = torch.arange(refs.numel(), device=refs.device, dtype=table.dtype)
    to[movers] = holes.to(table.dtype)
    for x in pools:
        x = x.view(x.shape[0], -1, page, *x.shape[2:])
        x[:, holes] = x[:, movers]
    mine = _held(table, length, page)
    table[mine] = to[table[mine].long()]
    refs[holes] = refs[movers]
    refs[movers] = 0
    used.fill_(u)


def _plain_pages(s):
    c = s["case"]
    t, n, refs, page = s["table"], s["len"], s["refs"], c["page"]
    if c["op"] == "fork":
        _plain_resize(t, n, refs, s["base"], s["ok"], page, s["cache"])
        _plain_fork(t, n, refs, s["parent"], page)
        _plain_resize(t, n, refs, s["grown"], s["ok"], page, s["cache"])
    else:
        s["now"].copy_(s["start"])
        _plain_compact(t, n, refs, s["used"], page, s["cache"])
    cu = s["cu"].long()
    row = torch.arange(s["rows"], device=t.device)
    b = torch.searchsorted(cu, row, right=True) - 1
    pos = s["at"].long()[b] - (cu[b + 1] - cu[b]) + row - cu[b]
    slots = t[b, pos // page].long() * page + pos % page
    return [s["cache"][2 * i][:, slots].float() * s["cache"][2 * i + 1][:, slots] for i in range(2)]


def _plain_attention(s):
    c = s["case"]
    b, h, g, hd = len(s["new"]), c["kv_heads"], c["heads"] // c["kv_heads"], c["hd"]
    nq, part = max(s["new"]), 512  # the sum over the keys in parts: a long one loses digits in 32 bits
    nk = -(-max(s["total"]) // part) * part
    dev = s["q"].device
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    i, j = torch.arange(nq, device=dev), torch.arange(nk, device=dev)
    rows = (s["cu"][:-1].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)  # [b, nq], padded
    page = (j // c["page"]).clamp(max=s["table"].shape[1] - 1)
    slots = s["table"].long().clamp(min=0)[:, page] * c["page"] + j % c["page"]  # [b, nk]
    k, v = ((s["cache"][2 * t][0][slots].float() * s["cache"][2 * t + 1][0][slots]).transpose(1, 2) for t in range(2))
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


def _plain_rope(s):
    c = s["case"]
    half, rot, kind = c["rot"] // 2, c["rot"], c["scaling"]
    m = _rope_settings(c)
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    theta = m["theta"] * (m["factor"] ** (rot / (rot - 2)) if kind == "base" else 1.0)
    f = theta ** (-2.0 * i / rot)
    if kind == "linear":
        f = f / m["factor"]
    if kind.startswith("ramp"):
        if kind == "ramp_turns":
            r = (m["trained"] * f / (2 * math.pi) - m["low"]) / (m["high"] - m["low"])
        else:
            at = [rot * math.log(m["trained"] / (2 * math.pi * n)) / (2 * math.log(theta)) for n in (m["high"], m["low"])]
            i0 = min(max(math.floor(at[0]), 0), half - 1)
            i1 = min(max(math.ceil(at[1]), 0), half - 1)
            r = 1 - (i - i0) / max(i1 - i0, 0.001)
        r = r.clamp(0, 1)
        f = f * (1 - r) / m["factor"] + f * r
    t = s["pos"].double()[:, None, None] * f
    cos, sin = ((fn(t) * m.get("gain", 1.0)).float() for fn in (torch.cos, torch.sin))
    out = []
    for x in (s["q"], s["k"]):
        a, b = (x[..., :half], x[..., half:rot]) if c["layout"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
        y = (a * cos - b * sin, a * sin + b * cos)
        y = torch.cat(y, -1) if c["layout"] == "half" else torch.stack(y, -1).flatten(-2)
        out.append(torch.cat([y, x[..., rot:]], -1))
    return out


def _plain_adapters(s):
    n = max(s["new"])
    cu, which = s["cu"].long(), s["which"].long()
    i = torch.arange(n, device="cuda")
    mine = i < (cu[1:] - cu[:-1])[:, None]
    x = s["x"][(cu[:-1, None] + i).clamp(max=s["x"].shape[0] - 1)]  # [seqs, n, cols], padded
    on = which >= 0
    scale = torch.where(on, s["scales"][which.clamp(min=0)], torch.zeros_like(s["scales"][:1]))[:, None, None]
    out = []
    for a, b, base in zip(s["a"], s["b"], s["base"]):
        a, b = a[which.clamp(min=0)].float(), b[which.clamp(min=0)].float()
        h = torch.matmul(x, a.transpose(1, 2).contiguous())
        y = torch.matmul(h, b.transpose(1, 2).contiguous()) * scale
        out.append(base + y[mine])
    return out


# ----------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    if not own:
        if c["kind"] == "rope":
            return dict(zip(("q", "k"), _plain_rope(s)))
        if c["kind"] == "adapters":
            return {"y": _plain_adapters(s)}
        if c["kind"] == "pages":
            k, v = _plain_pages(s)
            return {"table": s["table"], "len": s["len"], "refs": s["refs"], "ok": s["ok"], "used": s["used"],
                    "k": k, "v": v}
        return {"out": _plain_attention(s)}
    sh = s["stream"].cuda_stream
    if c["kind"] == "rope":
        s["rope"].apply_dev(s["pos"].data_ptr(), c["rows"], s["q"].data_ptr(), c["heads"], s["k"].data_ptr(),
                            c["kv_heads"], q_out_ptr=s["q_out"].data_ptr(), k_out_ptr=s["k_out"].data_ptr(), stream=sh)
        return {"q": s["q_out"], "k": s["k_out"]}
    if c["kind"] == "adapters":
        from welvet_amd.adapters import apply_dev
        apply_dev(s["sets"], s["batch"], s["x"].data_ptr(), [y.data_ptr() for y in s["y"]],
                  base_ptrs=[b.data_ptr() for b in s["base"]], stream=sh)
        return {"y": s["y"]}
    if c["kind"] == "pages":
        kv, t = s["kv"], s["tables"]
        if c["op"] == "fork":
            kv.resize_dev(t, s["base"].data_ptr(), s["ok"].data_ptr(), stream=sh)
            kv.fork_dev(t, s["parent"].data_ptr(), stream=sh)
            kv.resize_dev(t, s["grown"].data_ptr(), s["ok"].data_ptr(), stream=sh)
        else:
            with torch.cuda.stream(s["stream"]):
                s["now"].copy_(s["start"])
            kv.compact_dev(t, s["used"].data_ptr(), stream=sh)
        kv.slots_dev(s["batch"], s["slots"].data_ptr(), s["pos"].data_ptr(), stream=sh)
        for l in range(c["layers"]):
            kv.read_dev(l, s["slots"].data_ptr(), s["rows"], s["k"][l].data_ptr(), s["v"][l].data_ptr(), stream=sh)
        return {"table": s["table"], "len": s["len"], "refs": s["refs"], "ok": s["ok"], "used": s["used"],
                "k": s["k"], "v": s["v"]}
    s["kv"].attention_shared_dev(0, s["batch"], s["groups"], s["q"].data_ptr(), s["out"].data_ptr(), c["heads"],
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
    _, _, new, total = _share_plan(c)
    h, g, hd = c["kv_heads"], c["heads"] // c["kv_heads"], c["hd"]
    k, start = _share_rows(c, seed, 3, True)
    v, _ = _share_rows(c, seed, 4, False)
    q = _rows(seed, 5, sum(new), c["heads"], hd, False).double()
    out = torch.zeros_like(q)
    q0 = 0
    for b, (n, m) in enumerate(zip(new, total)):
        kk, vv = (_stored(x[start[b]:start[b] + m], c["type"]) for x in (k, v))
        pos = torch.arange(m - n, m, device="cuda")
        key = torch.arange(m, device="cuda")
        hide = key[None] > pos[:, None]
        if c["window"]:
            hide |= key[None] <= pos[:, None] - c["window"]
        for kh in range(h):
            kt, vt = kk[:, kh].t().contiguous(), vv[:, kh].contiguous()
            for qh in range(kh * g, kh * g + g):
                a = (q[q0:q0 + n, qh] @ kt) / math.sqrt(hd)
                out[q0:q0 + n, qh] = torch.softmax(a.masked_fill(hide, -math.inf), dim=1) @ vt
        q0 += n
    return out


def _exact_rope(c, seed):
    m, rot = _rope_settings(c), c["rot"]
    q, k, pos = _rope_inputs(c, seed)
    pos = pos.cpu().numpy().astype(np.float64)
    f = []
    for i in range(rot // 2):
        base = m["theta"]
        if c["scaling"] == "base":
            base = base * m["factor"] ** (rot / (rot - 2))
        w = math.pow(base, -2.0 * i / rot)
        if c["scaling"] == "linear":
            w /= m["factor"]
        elif c["scaling"] == "ramp_turns":
            turns = m["trained"] * w / (2 * math.pi)
            r = min(1.0, max(0.0, (turns - m["low"]) / (m["high"] - m["low"])))
            w = w * r + w / m["factor"] * (1 - r)
        elif c["scaling"] == "ramp_dims":
            ends = [rot / 2 * math.log(m["trained"] / (2 * math.pi * t)) / math.log(base) for t in (m["high"], m["low"])]
            lo, hi = max(0, math.floor(ends[0])), min(rot // 2 - 1, math.ceil(ends[1]))
            lo, hi = min(lo, rot // 2 - 1), max(hi, 0)
            r = min(1.0, max(0.0, 1 - (i - lo) / max(hi - lo, 0.001)))
            w = w * r + w / m["factor"] * (1 - r)
        f.append(w)
    angle = torch.from_numpy(pos[:, None] * np.array(f)[None]).cuda()
    turn = torch.polar(torch.full_like(angle, m.get("gain", 1.0)), angle)[:, None]
    out = []
    for x in (q, k):
        x = x.double()
        r = x[..., :rot].clone()
        if c["layout"] == "half":
            z = torch.complex(r[..., : rot // 2].contiguous(), r[..., rot // 2:].contiguous()) * turn
            r = torch.cat([z.real, z.imag], -1)
        else:
            r = torch.view_as_real(torch.view_as_complex(r.unflatten(-1, (rot // 2, 2)).contiguous()) * turn).flatten(-2)
        x[..., :rot] = r
        out.append(x)
    return out


def _exact_adapters(c, seed):
    new, which, _ = _adapt_plan(c)
    x, base, a, b, scales = _adapt_inputs(c, seed)
    out = [t.double() for t in base]
    at = 0
    for n, w in zip(new, which):
        for i in range(len(out) if w >= 0 else 0):
            h = x[at:at + n].double() @ a[i][w].double().t().contiguous()
            out[i][at:at + n] += scales[w] * (h @ b[i][w].double().t().contiguous())
        at += n
    return out


def _exact_pages(c, seed):
    """The rows that come back: those the sequences (fork: their group's parent) had before."""
    s = {}
    slots, old = _prepare_pages(s, c, seed)
    del slots
    _, n, _, _ = _page_plan(c)
    each = c["each"]
    if c["op"] == "fork":
        n = [n[i // each * each] for i in range(len(n))]
    start = np.concatenate([[0], np.cumsum(n)])
    of = s["parent"].cpu().numpy() if c["op"] == "fork" else np.arange(len(n))
    at = [start[of[i]] + n[i] - t + np.arange(t) for i, t in enumerate(s["back"])]
    at = _ints(np.concatenate(at), torch.int64)
    return [torch.stack([_stored(old[l][i][at], c["type"]) for l in range(c["layers"])]) for i in range(2)]


def exact(case, seed):
    c = case
    if c["kind"] == "rope":
        return dict(zip(("q", "k"), _exact_rope(c, seed)))
    if c["kind"] == "adapters":
        return {"y": _exact_adapters(c, seed)}
    if c["kind"] == "pages":
        k, v = _exact_pages(c, seed)
        return {"table": None, "len": None, "refs": None, "ok": None, "used": None, "k": k, "v": v}
    return {"out": _exact_attention(c, seed)}
