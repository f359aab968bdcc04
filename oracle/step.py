"""References for what a step does around the paged cache's attention (TEST
INFRASTRUCTURE ONLY): head norms and rotation by position, and the verification
of drafted tokens, in fp64 numpy from the definitions of include/kq_capi.h."""
from __future__ import annotations

import numpy as np


def rope(x, positions, freqs, weight=None, eps=1e-6, interleaved=False, factor=1.0):
    """x (T, H, D) normed and rotated, and per value the size that its roundings
    go by: the rotated pair's two values together, or the value itself."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    n = len(freqs)
    j = np.arange(n)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
    angle = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    cos, sin = np.cos(angle) * factor, np.sin(angle) * factor
    out, size = x.copy(), np.abs(x)
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(factor)
    return out, size


def verify_row(logits, drafts, u, draw, probs, temperature):
    """One row: logits (n, V), drafts (n - 1,), u (n,), probs (n, V) or None ->
    (accepted, token)."""
    n = len(logits)
    if n == 0:
        return 0, -1
    V = logits.shape[1]
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    for i in range(n):
        top = x[i].max()
        d = int(drafts[i]) if i < n - 1 else None
        known = d is not None and 0 <= d < V
        if not top > -np.inf:
            return i, -1
        if not temperature > 0:
            best = int(np.argmax(x[i]))
            if known and d == best:
                continue
            return i, best
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.exp((x[i] - top) / np.float64(temperature))
        e = np.where(x[i] > -np.inf, e, 0.0)
        Z = e.sum()
        q = None
        if probs is not None:
            q = np.asarray(probs[i], np.float64)
            q = np.where(np.isnan(q), 0.0, np.maximum(q, 0.0))
        if known and np.float64(u[i]) * (1.0 if q is None else q[d]) * Z < e[d]:
            continue
        w = e
        if d is not None:
            if q is not None:
                w = np.maximum(e - q * Z, 0.0)
            elif known:
                w = e.copy()
                w[d] = 0.0
            if not w.sum() > 0:
                w = e
        run = np.cumsum(w)
        over = np.nonzero((run > max(np.float64(draw), 0.0) * run[-1]) & (w > 0))[0]
        return i, int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])
    raise AssertionError("the last row ends it")


def verify(logits, tokens, cu, uniforms, draws, probs=None, temperature=1.0, kv_lens=None):
    """(accepted, tokens, keep_lens or None) of all rows; temperature a number or one a row."""
    acc, out, keep = [], [], []
    for b in range(len(cu) - 1):
        lo, hi = int(cu[b]), int(cu[b + 1])
        t = temperature if np.ndim(temperature) == 0 else temperature[b]
        a, v = verify_row(logits[lo:hi], tokens[lo + 1:hi], uniforms[lo:hi], draws[b],
                          None if probs is None else probs[lo:hi], t)
        acc.append(a)
        out.append(v)
        if kv_lens is not None:
            keep.append(max(int(kv_lens[b]) - (max(hi - lo, 1) - 1 - a), 0))
    return acc, out, keep if kv_lens is not None else None


def window_attention(q, k, v, n, scale, window, sinks, err=None, kv=None):
    """The last n of a row's kv keys (default: all of k) are its new tokens; token i
    sees the last `window` keys up to its own and the first `sinks`, of those that k
    holds: q (n, Hq, D), k / v (Hkv, keys, D) -> out (n, Hq, D) and the weighted
    mean of `err` (Hkv, keys, D; default |v|)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    err = np.abs(v) if err is None else np.asarray(err, np.float64)
    Hq, D = q.shape[1:]
    Hkv, have = k.shape[:2]
    kv = have if kv is None else kv
    out, far = np.zeros((len(q), Hq, D)), np.zeros((len(q), Hq, D))
    t = np.arange(have)
    for i in range(len(q)):
        me = kv - n + i
        see = (t <= me) & ((t > me - window) | (t < sinks))
        if not see.any():
            continue
        for h in range(Hkv):
            g = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            s = q[i, g] @ k[h, see].T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[i, g] = p @ v[h, see]
            far[i, g] = p @ err[h, see]
    return out, far
