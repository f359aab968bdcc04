"""The work that the paged KV cache's operators are measured on.

Three kinds of work, on a pool of pages [n_pages, Hkv, page_size, D] as a server keeps it:

  plan    block tables and slot maps of one step, built on the GPU from the requests' lengths: pages of rejected or
          finished tokens go back to the free stack, new tokens get theirs, every new token gets its slot
  write   new K / V rows into their slots, 16-bit or quantised to 8 bits in groups of 64, and (read) the rows at those
          slots read back, as a prefix is exported
  attend  the new tokens' attention over their rows' pages: one token a row, a verify block, a prompt chunk behind a
          context, and a batch that mixes them

A row's lengths follow from the case alone; pages are handed out in a random order; K, V and queries are N(0, 1), new
rows with a few large channels.  The plain forms are padded to the longest row, as a torch program without a kernel
would have them.
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a chat server's decode step: a few rows, one token each; launch latency
        dict(name="plan_decode_b8", kind="plan", B=8, ps=16, lo=200, hi=4000, mode="decode", n=1, lens=1),
        # a busy server's step: decode rows, verify blocks, prompt chunks, requests that ended, in one plan
        dict(name="plan_mixed_b300", kind="plan", B=300, ps=32, lo=1, hi=30000, mode="mixed", n=2048, lens=2),
        # the new tokens of a decode batch
        dict(name="write_decode_b32_bf16", kind="write", T=32, Hkv=8, D=128, ps=16, dtype="bf16", q8=False, read=False),
        # a prompt chunk of odd length stored, and its rows exported
        dict(name="write_read_4097_f16", kind="write", T=4097, Hkv=8, D=128, ps=64, dtype="f16", q8=False, read=True),
        # the same into an 8-bit cache
        dict(name="write_read_q8_2048_bf16", kind="write", T=2048, Hkv=8, D=128, ps=32, dtype="bf16", q8=True,
             read=True),
        # chat decode: three short rows, one layer's call
        dict(name="attend_decode_b3_bf16", kind="attend", mode="decode", B=3, n=1, Hq=32, Hkv=8, D=128, ps=16, lo=300,
             hi=1900, dtype="bf16", q8=False, lens=1),
        # a long-context batch with very different row lengths
        dict(name="attend_decode_b16_long_f16", kind="attend", mode="decode", B=16, n=1, Hq=32, Hkv=8, D=128, ps=64,
             lo=1024, hi=131072, dtype="f16", q8=False, lens=0),
        # decode over an 8-bit cache at moderate depth
        dict(name="attend_decode_q8_b6_bf16", kind="attend", mode="decode", B=6, n=1, Hq=32, Hkv=8, D=128, ps=32,
             lo=6000, hi=12000, dtype="bf16", q8=True, lens=2),
        # speculative verify: blocks of up to five tokens
        dict(name="attend_verify_b8_f16", kind="attend", mode="chunk", B=8, n=5, Hq=32, Hkv=8, D=128, ps=64, lo=2000,
             hi=8000, dtype="f16", q8=False, lens=3),
        # a full prefill chunk behind a context of 6000 tokens: the matrix cores' work
        dict(name="attend_chunk_2048_bf16", kind="attend", mode="decode", B=1, n=2048, Hq=32, Hkv=8, D=128, ps=64,
             lo=8048, hi=8048, dtype="bf16", q8=False, lens=4),
        # an odd chunk at head dim 256 over an 8-bit cache
        dict(name="attend_chunk_333_q8_d256_f16", kind="attend", mode="decode", B=1, n=333, Hq=16, Hkv=2, D=256, ps=32,
             lo=4200, hi=4200, dtype="f16", q8=True, lens=5),
        # chunked prefill beside decode: one prompt chunk, an idle row, the rest one token each
        dict(name="attend_mixed_b9_bf16", kind="attend", mode="mixed", B=9, n=500, Hq=32, Hkv=8, D=128, ps=16, lo=700,
             hi=6000, dtype="bf16", q8=False, lens=6),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "write", "write", "attend", "attend", "attend", "attend"])
    lens = rng.randrange(1 << 20)
    if kind == "plan":
        mode = rng.choice(["decode", "mixed", "chunk"])
        B = _log(rng, 1, 400)
        n = {"decode": 1, "mixed": _log(rng, 1, 2048), "chunk": _log(rng, 2, max(2, 60000 // B))}[mode]
        hi = _log(rng, 16, 100000)
        return dict(kind=kind, B=B, ps=rng.choice([16, 32, 64, 128]), lo=rng.choice([1, max(1, hi // 20), hi]), hi=hi,
                    mode=mode, n=n, lens=lens)
    dtype = rng.choice(["f16", "bf16"])
    q8 = rng.choice([False, False, True])
    D = rng.choice([64, 128, 128, 256, 512] if q8 else [64, 96, 128, 128, 256, 512])
    ps = rng.choice([16, 32, 64, 128, 256])
    if kind == "write":
        Hkv = rng.choice([1, 2, 4, 8])
        return dict(kind=kind, T=_log(rng, 1, 4096 * 1024 // (Hkv * D)), Hkv=Hkv, D=D, ps=ps, dtype=dtype, q8=q8,
                    read=rng.choice([False, True]) or q8)
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 4, 5, 8, 16])
    shape = rng.choice(["decode", "decode", "verify", "chunk", "chunk", "mixed"])
    if shape in ("decode", "verify"):
        B = _log(rng, 1, 32)
        n = 1 if shape == "decode" else rng.randrange(2, 9)
        hi = _log(rng, 16, max(32, min(131072, 400_000_000 // (B * Hkv * D), 200_000_000 // (B * n * Hq))))
        mode = "decode" if n == 1 else "chunk"
    else:
        B = _log(rng, 1, 6) if shape == "chunk" else _log(rng, 2, 12)
        n = _log(rng, 9, 2048)
        most = min(32768, 250_000_000 // (B * Hkv * D), 400_000_000 // (B * n * Hq), 60_000_000_000 // (B * n * Hq * D))
        n = min(n, max(9, most))
        hi = max(n, _log(rng, 16, max(32, most)))
        mode = shape
    return dict(kind=kind, mode=mode, B=B, n=n, Hq=Hq, Hkv=Hkv, D=D, ps=ps, lo=max(1, hi // rng.choice([1, 3, 20])),
                hi=hi, dtype=dtype, q8=q8, lens=lens)


# --------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _lens(case):
    """Host lengths of the case's rows: cached before the step, kept, new (plan); with the new ones, new (attend)."""
    r = np.random.default_rng(case["lens"])
    B, n = case["B"], case["n"]
    total = np.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"]), B)).round().astype(np.int64)
    if case["mode"] == "decode":
        new = np.full(B, n)
    elif case["mode"] == "chunk":
        new = r.integers(max(1, n // 2), n + 1, B)
    else:
        new = np.ones(B, np.int64)
        new[:1 + B // 64] = n
        if B >= 4:
            new[B // 2] = 0
    if case["kind"] == "attend":
        return np.maximum(total, new), new
    keep = total.copy()
    if case["mode"] == "mixed":
        keep = np.maximum(total - r.integers(0, 5, B) * (r.random(B) < 0.3), 0)  # rejected draft tokens
        ended = r.random(B) < 0.05
        keep[ended], new[ended] = 0, 0
    return total, keep, new


def _pages(n, ps):
    return -(-n // ps)


def _table(rows, ps, width, n_pages, gen):
    """A block table whose rows hold the pages of `rows` tokens in a random order, and the pages left over."""
    order = torch.randperm(n_pages, device="cuda", generator=gen).int()
    have = torch.tensor(_pages(rows, ps), device="cuda")
    first = have.cumsum(0) - have
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp(max=n_pages - 1)
    table = torch.where(col < have[:, None], order[at], 0).int().contiguous()
    return table, order[int(have.sum()):].contiguous()


def _rows(gen, *shape, dtype):
    x = torch.randn(*shape, device="cuda", generator=gen)
    big = torch.rand(shape[-1], device="cuda", generator=gen) < 0.02
    return (x * torch.where(big, 8.0, 1.0)).to(dtype)


def _pool(case, n_pages, gen):
    """K and V pools: [values] or [values, scales, biases], the values N(0, 1)."""
    dt, shape = DTYPE[case["dtype"]], (n_pages, case["Hkv"], case["ps"], case["D"])
    if not case["q8"]:
        return [[torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).to(dt)] for _ in range(2)]
    groups = (*shape[:3], case["D"] // 64)
    out = []
    for _ in range(2):
        step = (0.018 + 0.004 * torch.rand(*groups, device="cuda", generator=gen))
        out.append([torch.randint(0, 256, shape, device="cuda", generator=gen, dtype=torch.uint8), step.to(dt),
                    (step * -127.5).to(dt)])
    return out


def _plan_state(case, seed):
    gen = _gen(seed)
    total, keep, new = _lens(case)
    ps = case["ps"]
    width = int(_pages(np.maximum(total, keep + new), ps).max()) + 3
    used, want = int(_pages(total, ps).sum()), int(_pages(keep + new, ps).sum())
    n_pages = max(used, want) + used // 8 + 16
    table, left = _table(total, ps, width, n_pages, gen)
    free = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    free[:left.numel()] = left
    return dict(case=case, seq=_ints(total), keep=_ints(keep), new=_ints(new), table=table, free=free,
                count=_ints([left.numel()]), tokens=int(new.sum()))


def _write_state(case, seed):
    gen, T, ps = _gen(seed), case["T"], case["ps"]
    n_pages = _pages(T, ps) * 2 + 4
    k, v = _pool(case, n_pages, gen)
    x = [_rows(gen, T, case["Hkv"], case["D"], dtype=DTYPE[case["dtype"]]) for _ in range(2)]
    # the slots of a chunk: whole pages in a random order; of a decode batch: one in each of many pages
    page = torch.randperm(n_pages, device="cuda", generator=gen)[:_pages(T, ps)]
    slots = (page[:, None] * ps + torch.arange(ps, device="cuda")).reshape(-1)[:T].int().contiguous()
    return dict(case=case, k=k, v=v, x=x, slots=slots)


def _attend_state(case, seed):
    gen, ps = _gen(seed), case["ps"]
    kv, new = _lens(case)
    width = int(_pages(kv, ps).max())
    n_pages = int(_pages(kv, ps).sum()) + 8
    table, _ = _table(kv, ps, width, n_pages, gen)
    k, v = _pool(case, n_pages, gen)
    T = int(new.sum())
    q = torch.randn(T, case["Hq"], case["D"], device="cuda", generator=gen).to(DTYPE[case["dtype"]])
    return dict(case=case, q=q, k=k, v=v, table=table, kv_lens=_ints(kv), cu_q=_ints([0, *np.cumsum(new)]),
                max_q=int(new.max()), max_kv=int(kv.max()), scale=case["D"] ** -0.5)


def prepare(case, seed):
    return {"plan": _plan_state, "write": _write_state, "attend": _attend_state}[case["kind"]](case, seed)


# ----------------------------------------------------------- the plain forms

def _plan_plain(s):
    ps, T = s["case"]["ps"], s["tokens"]
    table, free, dev = s["table"], s["free"], s["seq"].device
    seq, new, count = s["seq"].long(), s["new"].long(), s["count"].long()
    base = torch.minimum(s["keep"].long(), seq)
    have, want = (seq + ps - 1) // ps, (base + new + ps - 1) // ps
    fits = want <= table.shape[1]
    give, take = (have - want).clamp(min=0), torch.where(fits, (want - have).clamp(min=0), 0)
    total = count + give.sum()
    first = take.cumsum(0) - take
    served = fits & ((take == 0) | (first + take <= total))
    left = total - (take * served).sum()
    kv = torch.where(served, base + new, seq)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), new.cumsum(0)])
    # the stack with the released pages on it
    col = torch.arange(table.shape[1], device=dev)
    stack = torch.arange(free.shape[0], device=dev)
    gone = (col >= want[:, None]) & (col < have[:, None])
    place = count + (give.cumsum(0) - give)[:, None] + col - want[:, None]
    spare = free.shape[0]
    full = torch.cat([free, free.new_zeros(1)])
    full.scatter_(0, torch.where(gone, place, spare).reshape(-1), table.reshape(-1))
    full = full[:spare]
    # tokens
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = base[b] + t - cu[b]
    nth = pos // ps
    fresh = full[(total - 1 - (first[b] + nth - have[b])).clamp(0, spare - 1)]
    page = torch.where(nth < have[b], table[b, nth.clamp(max=table.shape[1] - 1)], fresh).long()
    slots = torch.where(served[b], page * ps + pos % ps, -1).int()
    pos = torch.where(served[b], pos, -1).int()
    # state
    add = (col >= have[:, None]) & (col < want[:, None]) & served[:, None]
    pick = (total - 1 - (first[:, None] + col - have[:, None])).clamp(0, spare - 1)
    table.copy_(torch.where(add, full[pick], table))
    free.copy_(torch.where((stack >= count) & (stack < left), full, free))
    return dict(cu_q=cu.int(), kv_lens=kv.int(), slots=slots, positions=pos, free_count=left.int(),
                refused=(~served).int(), table=table, free=free)


def _quantise(x, dt):
    g = x.float().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, b = ((hi - lo) / 255).to(dt), lo.to(dt)
    q = ((g - b.float()) / s.float()).round().clamp(0, 255)
    q = torch.where(s == 0, 0, q).to(torch.uint8)
    return [q.flatten(-2), s.squeeze(-1), b.squeeze(-1)]


def _values(pool):
    """Pool rows as 32-bit values."""
    if len(pool) == 1:
        return pool[0].float()
    q, s, b = pool
    return (q.float().unflatten(-1, (-1, 64)) * s.float()[..., None] + b.float()[..., None]).flatten(-2)


def _write_plain(s):
    case = s["case"]
    dt = DTYPE[case["dtype"]]
    ok = s["slots"] >= 0
    slot = s["slots"][ok].long()
    page, off = slot // case["ps"], slot % case["ps"]
    out = {}
    for name, pool, x in (("k", s["k"], s["x"][0]), ("v", s["v"], s["x"][1])):
        for dst, rows in zip(pool, _quantise(x[ok], dt) if case["q8"] else [x[ok]]):
            dst[page, :, off] = rows
        out[name] = pool[1:] if case["q8"] else pool
        if case["read"]:
            got = _values([t[page, :, off] for t in pool]).to(dt)
            out["read_" + name] = torch.where(ok[:, None, None], got, 0)
    return out


def _attend_plain(s):
    case = s["case"]
    B, Hkv, D, G = case["B"], case["Hkv"], case["D"], case["Hq"] // case["Hkv"]
    T, mq = s["q"].shape[0], s["max_q"]
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    new = cu[1:] - cu[:-1]
    at = s["table"].long()
    keys, vals = (_values([t[at] for t in pool]).transpose(1, 2).reshape(B, Hkv, -1, D) for pool in (s["k"], s["v"]))
    i = torch.arange(mq, device=cu.device)
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"][rows].float().view(B, mq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * mq, D)
    score = torch.matmul(q * s["scale"], keys.transpose(2, 3)).view(B, Hkv, G, mq, -1)
    last = kv[:, None] - new[:, None] + i  # the last key that token i of each row sees
    seen = torch.arange(score.shape[-1], device=cu.device) <= last[:, :, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = torch.where(seen[:, None, None], p, 0)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hkv, G * mq, -1), vals).view(B, Hkv, G, mq, D) / total.clamp(min=1e-30)
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return out.permute(0, 3, 1, 2, 4).reshape(B, mq, Hkv * G, D)[b, t - cu[b]].to(s["q"].dtype)


# ----------------------------------------------------------------- one pass

def _own(s):
    from gmlx_amd import ops
    case = s["case"]
    if case["kind"] == "plan":
        p = ops.paged_plan(s["seq"], s["new"], s["table"], s["free"], s["count"], case["ps"], s["tokens"],
                           keep_lens=s["keep"])
        return dict(cu_q=p.cu_q, kv_lens=p.kv_lens, slots=p.slots, positions=p.positions, free_count=p.free_count,
                    refused=p.refused, table=s["table"], free=s["free"])
    scales = {}
    if case["q8"]:
        scales = dict(k_scales=s["k"][1], k_biases=s["k"][2], v_scales=s["v"][1], v_biases=s["v"][2])
    if case["kind"] == "attend":
        return ops.sdpa_paged(s["q"], s["k"][0], s["v"][0], s["table"], s["kv_lens"], s["cu_q"], s["scale"],
                              max_q=s["max_q"], max_kv=s["max_kv"], **scales)
    ops.paged_write(s["x"][0], s["x"][1], s["k"][0], s["v"][0], s["slots"], **scales)
    out = dict(k=s["k"][1:] if case["q8"] else s["k"], v=s["v"][1:] if case["q8"] else s["v"])
    if case["read"]:
        out["read_k"], out["read_v"] = ops.paged_read(s["k"][0], s["v"][0], s["slots"], **scales)
    return out


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan_plain, "write": _write_plain, "attend": _attend_plain}[state["case"]["kind"]](state)


# --------------------------------------------------------------------- work

def _row_bytes(case):
    """Bytes of one token's K and V over the kv heads."""
    D = case["D"]
    return 2 * case["Hkv"] * (D + D // 64 * 4 if case["q8"] else 2 * D)


def work(case):
    if case["kind"] == "plan":
        total, keep, new = _lens(case)
        have, want = _pages(total, case["ps"]), _pages(keep + new, case["ps"])
        moved = int(np.abs(have - want).sum())
        return {"bytes": 4 * (6 * case["B"] + 3 * int(new.sum()) + 2 * moved), "flops": 0}
    if case["kind"] == "write":
        rows = case["T"] * 2 * case["Hkv"] * case["D"] * 2
        kept = case["T"] * _row_bytes(case)
        return {"bytes": 4 * case["T"] + rows + kept + (kept + rows + 4 * case["T"] if case["read"] else 0), "flops": 0}
    kv, new = _lens(case)
    seen = int((new * kv - new * (new - 1) // 2).sum())
    used = int(kv[new > 0].sum())
    return {"bytes": used * _row_bytes(case) + 4 * int(new.sum()) * case["Hq"] * case["D"],
            "flops": 4 * case["Hq"] * case["D"] * seen}


# --------------------------------------------------------------------- exact

def _exact_rows(pool, table, n, ps):
    """Row values [Hkv, n, D] of the first n tokens of a block table row, in 64 bits."""
    t = torch.arange(n, device=table.device)
    got = [x[table[t // ps].long(), :, t % ps].double() for x in pool]
    if len(got) == 3:
        q, sc, bi = got
        got = [q * sc.repeat_interleave(64, -1) + bi.repeat_interleave(64, -1)]
    return got[0].transpose(0, 1)


def _attend_exact(case, seed):
    s = _attend_state(case, seed)
    kv, new = _lens(case)
    G, out, at = case["Hq"] // case["Hkv"], torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b in range(case["B"]):
        n, L = int(new[b]), int(kv[b])
        if not n:
            continue
        k, v = (_exact_rows(p, s["table"][b], L, case["ps"]) for p in (s["k"], s["v"]))
        hidden = torch.arange(L, device="cuda") > torch.arange(L - n, L, device="cuda")[:, None]
        for h in range(case["Hq"]):
            w = s["q"][at:at + n, h].double() @ k[h // G].T * s["scale"]
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h] = w @ v[h // G]
        at += n
    return out


def _write_exact(case, seed):
    s = _write_state(case, seed)
    dt, out = DTYPE[case["dtype"]], {}
    page, off = s["slots"].long() // case["ps"], s["slots"].long() % case["ps"]
    for name, pool, x in (("k", s["k"], s["x"][0]), ("v", s["v"], s["x"][1])):
        if case["q8"]:
            g = x.double().view(*x.shape[:2], -1, 64)
            low = g.min(-1).values
            step = ((g.max(-1).values - low) / 255).to(dt).double()
            low = low.to(dt).double()
            q = torch.round((g - low[..., None]) / step[..., None]).clamp(0, 255)
            kept = [None, step, low]
            rows = (q * step[..., None] + low[..., None]).view(x.shape)
        else:
            kept, rows = [x.double()], x.double()
        held = [p.double() for p in pool]
        for dst, new in zip(held, kept):
            if new is not None:
                dst[page, :, off] = new
        out[name] = held[1:] if case["q8"] else held
        if case["read"]:
            out["read_" + name] = rows
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    return (_attend_exact if case["kind"] == "attend" else _write_exact)(case, seed)
