"""The paged KV cache and its attention in float64 numpy: what a row is held
as, and causal attention over held rows, with bounds on what fp16 pairs and
f32 sums may be off by."""
import numpy as np

LOG2E = 1.4426950408889634


def stored(x, typ):
    """The values that the cache holds of rows x[..., hd] (float32)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(x).max(-1, keepdims=True)
        y = x.astype(np.float64)
        if typ == "f16":
            s = np.ldexp(1.0, np.frexp(np.where(np.isfinite(amax), amax, 1.0).astype(np.float64))[1] - 15)
            out = (y / s).astype(np.float16).astype(np.float64) * s
        else:
            s = (amax / np.float32(127)).astype(np.float64)
            t = y / np.where(s > 0, s, 1.0)
            out = np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -127, 127) * s
        out = np.where(amax < 2.0 ** -100, 0.0, out)
        return np.where(np.isfinite(x).all(-1, keepdims=True), out, np.nan).astype(np.float32).astype(np.float64)


def attention(q, k, v, n, scale, window=0, present=None):
    """q [n, H, hd] of one sequence's new tokens over its keys k, v [L, KV, hd]
    (held values). present [L]: keys whose page exists. Returns the rows and a
    bound on each value's error: scores are off by at most
    d = (2^-21 + (hd + 2) 2^-24) scale sum|q k| (fp16 pairs, then hd products
    summed in f32 and two scales), each exponential by a relative d + 2^-21,
    the sums over L keys by L 2^-24 and their quotient by as much again. The
    fp16 pair of P_j = 2^14 p_j s_j 2^-E (2^E at most twice the largest scale)
    also has an absolute error of 2^-25, half the smallest step of its second
    term: 2^-39 2^E |c_j| in the sum of p_j V_j, so at most 2^-37 max |V| a key
    (|c_j| scale <= 2 max |V| with fp16 codes), over a sum of p that is >= 1."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    H, hd, L = q.shape[1], q.shape[2], k.shape[0]
    G = H // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    pos = L - n + np.arange(n)[:, None]
    key = np.arange(L)[None]
    seen = key <= pos
    if window > 0:
        seen &= key > pos - window
    if present is not None:
        seen &= np.asarray(present, bool)[None]
    for h in range(H if n and L else 0):
        kk, vv = k[:, h // G], v[:, h // G]
        s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
        m = np.max(s, 1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
        p = np.where(seen, p, 0.0)
        l = p.sum(1, keepdims=True)
        w = p / np.where(l > 0, l, 1.0)
        out[:, h] = w @ np.where(seen.any(0)[:, None], vv, 0.0)
        big = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T * abs(scale), 0.0).max(1, keepdims=True)
        d = (2.0 ** -21 + (hd + 2) * 2.0 ** -24) * big + 2.0 ** -21 + L * 2.0 ** -24
        tol[:, h] = 2 * d * (w @ np.where(seen.any(0)[:, None], np.abs(vv), 0.0)) + L * 2.0 ** -37 * np.where(
            seen.any(0)[:, None], np.abs(vv), 0.0).max(initial=0.0) + 1e-30
    return out, tol
