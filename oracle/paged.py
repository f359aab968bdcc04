"""Paged KV cache reference (TEST INFRASTRUCTURE ONLY): the plan in plain
Python, the 8-bit affine quantiser and the attention of new tokens in fp64
numpy, from the definitions of include/kq_capi.h."""
from __future__ import annotations

import numpy as np


def plan(seq, new, table, stack, count, page, max_tokens, keep=None):
    """(cu_q, kv_lens, slots, positions, free_count, refused) and the table and
    stack after the step, all as new arrays / lists."""
    B, width = table.shape
    table, stack = table.copy(), list(int(x) for x in stack)
    count = min(max(int(count), 0), len(stack))
    seq = [min(max(int(s), 0), width * page) for s in seq]
    new = [max(int(n), 0) for n in new]
    base = [min(max(int(k), 0), s) for k, s in zip(keep, seq)] if keep is not None else list(seq)
    have = [-(-s // page) for s in seq]
    want = [-(-(b + n) // page) for b, n in zip(base, new)]
    free = stack[:count]
    for b in range(B):
        free += [int(x) for x in table[b, want[b]:have[b]]]
    free = free[:len(stack)]
    pages = [list(table[b, :have[b]]) for b in range(B)]
    short, refused, kv = False, [0] * B, []
    for b in range(B):
        need = max(want[b] - have[b], 0)
        if want[b] > width or (need and (short or need > len(free))):
            # (a row too wide for the table takes nothing from the stack's count)
            short |= want[b] <= width
            refused[b] = 1
            kv.append(seq[b])
            continue
        for j in range(need):
            pages[b].append(free.pop())
            table[b, have[b] + j] = pages[b][-1]
        kv.append(base[b] + new[b])
    for i in range(count, len(free)):
        stack[i] = free[i]
    slots, pos = [], []
    for b in range(B):
        for i in range(new[b]):
            p = base[b] + i
            pos.append(-1 if refused[b] else p)
            slots.append(-1 if refused[b] else int(pages[b][p // page]) * page + p % page)
    pad = max(0, max_tokens - len(slots))
    cu = np.concatenate([[0], np.cumsum(new)])
    return (cu, kv, (slots + [-1] * pad)[:max_tokens], (pos + [-1] * pad)[:max_tokens], len(free), refused, table,
            stack)


def attention(q, k, v, n, scale, err=None):
    """The last n of the row's len(k[0]) keys are its new tokens: q (n, Hq, D),
    k / v (Hkv, kv, D) -> out (n, Hq, D) and the weighted mean of `err` (Hkv,
    kv, D; default |v|) under the same probabilities, fp64."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    err = np.abs(v) if err is None else np.asarray(err, np.float64)
    Hq, D = q.shape[1:]
    Hkv, kv = k.shape[:2]
    out, far = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    for i in range(n):
        L = kv - n + i + 1
        if L <= 0:
            continue
        for h in range(Hkv):
            G = Hq // Hkv
            s = q[i, h * G:(h + 1) * G] @ k[h, :L].T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[i, h * G:(h + 1) * G] = p @ v[h, :L]
            far[i, h * G:(h + 1) * G] = p @ err[h, :L]
    return out, far
