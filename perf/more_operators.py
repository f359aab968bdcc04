"""The work that the operators around a step of the paged cache are measured on.

Three kinds of work, as a server does them in every layer or at every step:

  rope    queries and keys normed for each head and rotated by their positions, in one pass; or the same with the keys
          and values going straight to their slots of a paged cache, 16-bit or 8-bit
  attend  the new tokens' attention over a paged cache, where a token sees the last `window` keys and the row's first
          `sinks`; pages between them have been given back (their block table entries are -1)
  verify  drafted tokens against the target's logits: how many of each row stand, and the token after them, from given
          random numbers, with or without the probabilities that the drafts were drawn from

A row's lengths follow from the case alone.  Queries, keys and values are N(0, 1), logits have a few likely tokens above
a broad rest, drafts are drawn from a model that is near the target.  The plain forms are padded to the longest row, as
a torch program without a kernel would have them.
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one chat, one token: the smallest call, launch latency
        dict(name="rope_write_b1_bf16", kind="rope", T=1, Hq=32, Hkv=8, D=128, R=128, pairs="half", norm=True, far=8000,
             write=True, q8=False, ps=16, dtype="bf16"),
        # a decode batch into an 8-bit cache, a quarter of the head rotated, long contexts
        dict(name="rope_write_q8_b37_f16", kind="rope", T=37, Hq=16, Hkv=2, D=256, R=64, pairs="half", norm=True,
             far=1000000, write=True, q8=True, ps=32, dtype="f16"),
        # a prompt chunk, queries and keys normed and rotated
        dict(name="rope_2048_bf16", kind="rope", T=2048, Hq=32, Hkv=8, D=128, R=128, pairs="half", norm=True, far=40000,
             write=False, q8=False, ps=16, dtype="bf16"),
        # a chunk of odd length into the cache, neighbours paired, no norm
        dict(name="rope_write_4097_f16", kind="rope", T=4097, Hq=32, Hkv=8, D=128, R=128, pairs="next", norm=False,
             far=131072, write=True, q8=False, ps=64, dtype="f16"),
        # a small decode batch behind long contexts
        dict(name="window_decode_b5_bf16", kind="attend", mode="decode", B=5, n=1, Hq=32, Hkv=8, D=128, ps=16, lo=900,
             hi=60000, window=1024, sinks=4, dtype="bf16", q8=False, lens=1),
        # a large one over an 8-bit cache
        dict(name="window_decode_q8_b48_f16", kind="attend", mode="decode", B=48, n=1, Hq=32, Hkv=8, D=128, ps=64,
             lo=1000, hi=200000, window=4096, sinks=64, dtype="f16", q8=True, lens=2),
        # a full prefill chunk behind a context of 20000: the matrix cores' work
        dict(name="window_chunk_2048_bf16", kind="attend", mode="decode", B=1, n=2048, Hq=32, Hkv=8, D=128, ps=64,
             lo=22048, hi=22048, window=2000, sinks=4, dtype="bf16", q8=False, lens=3),
        # chunked prefill beside decode at head dim 256, a window that ends inside tiles
        dict(name="window_mixed_b9_f16", kind="attend", mode="mixed", B=9, n=500, Hq=16, Hkv=4, D=256, ps=32, lo=700,
             hi=9000, window=777, sinks=1, dtype="f16", q8=False, lens=4),
        # one chat, three drafted tokens, greedy
        dict(name="verify_greedy_b1", kind="verify", B=1, k=3, V=32000, dtype="bf16", probs="none", temp=0.0, lens=1),
        # a batch whose drafts were looked up, not drawn
        dict(name="verify_b16_k4_bf16", kind="verify", B=16, k=4, V=131072, dtype="bf16", probs="none", temp=0.7, lens=2),
        # drafts drawn from a small model, an odd vocabulary, 32-bit logits
        dict(name="verify_probs_b7_f32", kind="verify", B=7, k=5, V=50001, dtype="f32", probs="f32", temp=1.0, lens=3),
        # a busy server: many rows of ragged drafts over a large vocabulary
        dict(name="verify_probs_b96_f16", kind="verify", B=96, k=4, V=152064, dtype="f16", probs="f32", temp=0.8, lens=4),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "attend", "attend", "attend", "verify", "verify"])
    lens = rng.randrange(1 << 20)
    if kind == "verify":
        V, dtype = _log(rng, 250, 160000), rng.choice(["f16", "bf16", "bf16", "f32"])
        k = rng.randrange(0, 9)
        probs = rng.choice(["none", "f32", "f32", dtype]) if k else "none"
        B = _log(rng, 1, max(1, min(128, 60_000_000 // (V * (k + 1)))))
        return dict(kind=kind, B=B, k=k, V=V, dtype=dtype, probs=probs, temp=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5]),
                    lens=lens)
    dtype = rng.choice(["f16", "bf16"])
    q8 = rng.choice([False, False, True])
    D = rng.choice([64, 128, 128, 256, 512] if q8 else [64, 96, 128, 128, 256, 512])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 4, 5, 8, 16])
    ps = rng.choice([16, 32, 64, 128, 256])
    if kind == "rope":
        write = rng.choice([False, True, True]) or q8
        R = 16 * rng.choice([D // 16, D // 16, rng.randrange(1, D // 16 + 1)])
        return dict(kind=kind, T=_log(rng, 1, 4097 * 40 * 128 // ((Hq + 2 * Hkv) * D)), Hq=Hq, Hkv=Hkv, D=D, R=R,
                    pairs=rng.choice(["half", "half", "next"]), norm=rng.choice([True, False]), far=_log(rng, 4, 1000000),
                    write=write, q8=q8, ps=ps, dtype=dtype)
    shape = rng.choice(["decode", "decode", "verify", "chunk", "chunk", "mixed"])
    window, sinks = _log(rng, 1, 8192), rng.choice([0, 0, 1, 4, 4, 16, 130])
    if shape in ("decode", "verify"):
        n = 1 if shape == "decode" else rng.randrange(2, 9)
        B = _log(rng, 1, max(1, min(64, 200_000_000 // ((window + sinks + n) * n * Hq), 400_000_000 // ((window + sinks) * Hkv * D))))
        mode = "decode" if n == 1 else "chunk"
    else:
        B = _log(rng, 1, 6) if shape == "chunk" else _log(rng, 2, 12)
        n = _log(rng, 9, 2048)
        most = min(250_000_000 // (B * Hkv * D), 400_000_000 // (B * n * Hq), 60_000_000_000 // (B * n * Hq * D))
        window = max(1, min(window, most - n))
        n = min(n, max(9, most))
        mode = shape
    hi = max(n, _log(rng, 16, 200000))
    return dict(kind=kind, mode=mode, B=B, n=n, Hq=Hq, Hkv=Hkv, D=D, ps=ps, lo=max(1, hi // rng.choice([1, 3, 20])), hi=hi,
                window=window, sinks=sinks, dtype=dtype, q8=q8, lens=lens)


# --------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _pages(n, ps):
    return -(-n // ps)


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


def _freqs(R):
    """Radians a position of the R / 2 pairs, in 64 bits."""
    return 500000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)


def _rope_state(case, seed):
    gen, T, ps, D, dt = _gen(seed), case["T"], case["ps"], case["D"], DTYPE[case["dtype"]]
    Hq, Hkv = case["Hq"], case["Hkv"]
    packed = _rows(gen, T, Hq + 2 * Hkv, D, dtype=dt)  # a layer's q | k | v product
    s = dict(case=case, q=packed[:, :Hq], k=packed[:, Hq:Hq + Hkv], v=packed[:, Hq + Hkv:], freqs=_freqs(case["R"]))
    s["positions"] = torch.randint(0, case["far"], (T,), device="cuda", generator=gen, dtype=torch.int32)
    s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(D, device="cuda", generator=gen)).to(dt) for _ in range(2))
    if case["write"]:
        n_pages = _pages(T, ps) * 2 + 4
        s["pools"] = _pool(case, n_pages, gen)
        page = torch.randperm(n_pages, device="cuda", generator=gen)[:_pages(T, ps)]
        s["slots"] = (page[:, None] * ps + torch.arange(ps, device="cuda")).reshape(-1)[:T].int().contiguous()
    return s


def _lens(case):
    """Host lengths of an attention case's rows: cached with the new tokens, new."""
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
    return np.maximum(total, new), new


def _attend_state(case, seed):
    gen, ps = _gen(seed), case["ps"]
    kv, new = _lens(case)
    # a row holds the pages of its first keys and of those that its first new token's window reaches
    col = np.arange(int(_pages(kv, ps).max()))
    first = np.maximum(kv - new + 1 - case["window"], 0) // ps
    held = ((col < _pages(case["sinks"], ps)) | (col >= first[:, None])) & (col < _pages(kv, ps)[:, None])
    n_pages = int(held.sum()) + 8
    order = torch.randperm(n_pages, device="cuda", generator=gen).int()
    table = torch.full(held.shape, -1, dtype=torch.int32, device="cuda")
    table[torch.tensor(held, device="cuda")] = order[:int(held.sum())]
    k, v = _pool(case, n_pages, gen)
    T = int(new.sum())
    q = torch.randn(T, case["Hq"], case["D"], device="cuda", generator=gen).to(DTYPE[case["dtype"]])
    return dict(case=case, q=q, k=k, v=v, table=table, kv_lens=_ints(kv), cu_q=_ints([0, *np.cumsum(new)]),
                max_q=int(new.max()), max_kv=int(kv.max()), scale=case["D"] ** -0.5)


def _drafts(case):
    """Drafted tokens of each row: all of k for half the rows, fewer for the others."""
    r = np.random.default_rng(case["lens"])
    return np.where(r.random(case["B"]) < 0.5, case["k"], r.integers(0, case["k"] + 1, case["B"]))


def _verify_state(case, seed):
    gen, V, temp = _gen(seed), case["V"], case["temp"]
    n = _drafts(case) + 1
    T, B = int(n.sum()), case["B"]
    logits = 2.0 * torch.randn(T, V, device="cuda", generator=gen)
    likely = torch.randint(0, V, (T, 8), device="cuda", generator=gen)
    logits.scatter_add_(1, likely, 12 + 2.0 * torch.randn(T, 8, device="cuda", generator=gen))
    logits = logits.to(DTYPE[case["dtype"]])
    near = logits.float() + 0.6 * torch.randn(T, V, device="cuda", generator=gen)
    near.div_(max(temp, 0.25))
    noise = torch.rand(T, V, device="cuda", generator=gen).clamp_(min=1e-20).log_().neg_().log_().neg_()
    nxt = (near + noise).argmax(1)  # drawn from the softmax of `near`
    del noise
    tokens = torch.zeros(T, dtype=torch.int32, device="cuda")
    tokens[1:] = nxt[:-1].int()  # the draft after row t is what row t + 1 was fed
    s = dict(case=case, logits=logits, tokens=tokens, cu=_ints([0, *np.cumsum(n)]), n=int(n.max()),
             u=torch.rand(T, device="cuda", generator=gen), draws=torch.rand(B, device="cuda", generator=gen),
             kv_lens=_ints(n + 100), probs=None)
    if case["probs"] != "none":
        s["probs"] = torch.softmax(near, 1).to(DTYPE[case["probs"]])
    return s


def prepare(case, seed):
    return {"rope": _rope_state, "attend": _attend_state, "verify": _verify_state}[case["kind"]](case, seed)


# ----------------------------------------------------------- the plain forms

def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, s):
    case = s["case"]
    R = case["R"]
    angle = s["positions"].double()[:, None] * s["freqs"]
    cos, sin = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))
    if case["pairs"] == "half":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., R:]], -1)


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


def _stored(pool, rows, s):
    """`rows` in their slots of a pool: the pool, or what an 8-bit pool then holds there."""
    case = s["case"]
    page, off = s["slots"].long() // case["ps"], s["slots"].long() % case["ps"]
    dt = DTYPE[case["dtype"]]
    if not case["q8"]:
        pool[0][page, :, off] = rows
        return pool[0]
    q, sc, bi = _quantise(rows, dt)
    pool[0][page, :, off], pool[1][page, :, off], pool[2][page, :, off] = q, sc, bi
    return _values([t[page, :, off] for t in pool]).to(dt)


def _rope_plain(s):
    case = s["case"]
    q, k = s["q"].float(), s["k"].float()
    if case["norm"]:
        q, k = _normed(q, s["wq"]), _normed(k, s["wk"])
    q, k = (_rotated(x, s).to(s["q"].dtype) for x in (q, k))
    if not case["write"]:
        return dict(q=q, k=k)
    return dict(q=q, k=_stored(s["pools"][0], k, s), v=_stored(s["pools"][1], s["v"], s))


def _attend_plain(s):
    case = s["case"]
    B, Hkv, D, G, ps = case["B"], case["Hkv"], case["D"], case["Hq"] // case["Hkv"], case["ps"]
    T, mq, W, S = s["q"].shape[0], s["max_q"], case["window"], case["sinks"]
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    new = cu[1:] - cu[:-1]
    # the keys that some token of a row sees: the first ones, then from where its first token's window begins
    low = (kv - new + 1 - W).clamp(min=0)
    skipped = (low - S).clamp(min=0)
    j = torch.arange(min(s["max_kv"], S + W + mq), device=cu.device)
    key = torch.where(j < S, j, j + skipped[:, None])
    at = s["table"].long().gather(1, (key // ps).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    keys, vals = (_values([t[at, :, key % ps] for t in pool]).transpose(1, 2) for pool in (s["k"], s["v"]))
    i = torch.arange(mq, device=cu.device)
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"][rows].float().view(B, mq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * mq, D)
    score = torch.matmul(q * s["scale"], keys.transpose(2, 3).contiguous()).view(B, Hkv, G, mq, -1)
    last = (kv[:, None] - new[:, None] + i)[:, :, None]  # token i's own key
    key = key[:, None]
    seen = (key <= last) & ((key > last - W) | (key < S))
    seen = seen[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = torch.where(seen, p, 0)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hkv, G * mq, -1), vals.contiguous()).view(B, Hkv, G, mq, D) / total.clamp(min=1e-30)
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return out.permute(0, 3, 1, 2, 4).reshape(B, mq, Hkv * G, D)[b, t - cu[b]].to(s["q"].dtype)


def _verify_plain(s):
    case, cu, temp = s["case"], s["cu"].long(), s["case"]["temp"]
    B, V, T, n = case["B"], case["V"], s["logits"].shape[0], cu[1:] - cu[:-1]
    b = torch.arange(B, device=cu.device)
    x = s["logits"]
    following = torch.cat([s["tokens"][1:], s["tokens"][:1]]).long()  # the draft that row t is asked about
    top = x.float().argmax(1)
    if temp == 0:
        stands = following == top
    else:
        x = x.double()
        e = torch.exp((x - x.amax(1, keepdim=True)) / temp)
        total = e.sum(1)
        q = 1.0 if s["probs"] is None else s["probs"].gather(1, following[:, None])[:, 0].double()
        stands = s["u"].double() * q * total < e.gather(1, following[:, None])[:, 0]
    i = torch.arange(s["n"], device=cu.device)
    fails = ~stands[(cu[:-1, None] + i).clamp(max=T - 1)] | (i >= n[:, None] - 1)  # (the last row's is no draft)
    accepted = fails.int().argmax(1)
    row = cu[:-1] + accepted
    if temp == 0:
        token = top[row]
    else:
        w = e[row]
        if s["probs"] is not None:
            rest = (w - s["probs"][row].double() * total[row, None]).clamp(min=0)
        else:
            rest = w.scatter(1, following[row][:, None], 0.0)
        refused = (accepted < n - 1) & (rest.sum(1) > 0)
        w = torch.where(refused[:, None], rest, w)
        run = w.cumsum(1)
        token = (run > s["draws"].double()[:, None] * run[:, -1:]).int().argmax(1)
    return dict(accepted=accepted.int(), token=token.int(), keep=(s["kv_lens"].long() - n + 1 + accepted).int())


# ----------------------------------------------------------------- one pass

def _scales(k, v):
    return dict(k_scales=k[1], k_biases=k[2], v_scales=v[1], v_biases=v[2]) if len(k) == 3 else {}


def _own(s):
    from gmlx_amd import ops
    case = s["case"]
    if case["kind"] == "verify":
        r = ops.verify_drafts(s["logits"], s["tokens"], s["cu"], s["u"], s["draws"], draft_probs=s["probs"],
                              temperature=case["temp"], kv_lens=s["kv_lens"])
        return dict(accepted=r.accepted, token=r.tokens, keep=r.keep_lens)
    if case["kind"] == "attend":
        return ops.sdpa_paged(s["q"], s["k"][0], s["v"][0], s["table"], s["kv_lens"], s["cu_q"], s["scale"],
                              max_q=s["max_q"], max_kv=s["max_kv"], window=case["window"], sinks=case["sinks"],
                              **_scales(s["k"], s["v"]))
    turn = dict(interleaved=case["pairs"] == "next")
    if case["norm"]:
        turn.update(q_weight=s["wq"], k_weight=s["wk"], eps=EPS)
    if not case["write"]:
        q, k = ops.rope_qk(s["q"], s["k"], s["positions"], s["freqs"], **turn)
        return dict(q=q, k=k)
    k, v = s["pools"]
    q = ops.paged_write_rope(s["q"], s["k"], s["v"], k[0], v[0], s["slots"], s["positions"], s["freqs"], **_scales(k, v),
                             **turn)
    if case["q8"]:
        k, v = ops.paged_read(k[0], v[0], s["slots"], **_scales(k, v))
        return dict(q=q, k=k, v=v)
    return dict(q=q, k=k[0], v=v[0])


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope_plain, "attend": _attend_plain, "verify": _verify_plain}[state["case"]["kind"]](state)


# --------------------------------------------------------------------- work

def _row_bytes(case):
    """Bytes of one token's K and V over the kv heads."""
    D = case["D"]
    return 2 * case["Hkv"] * (D + D // 64 * 4 if case["q8"] else 2 * D)


def work(case):
    if case["kind"] == "rope":
        T, D, Hq, Hkv = case["T"], case["D"], case["Hq"], case["Hkv"]
        moved = 2 * T * 2 * D * (Hq + Hkv) + 4 * T
        if case["write"]:
            moved = T * (2 * 2 * D * Hq + 2 * 2 * D * Hkv + _row_bytes(case) + 8)
            if case["q8"]:
                moved += T * (_row_bytes(case) + 4 * D * Hkv + 4)
        return {"bytes": moved, "flops": 6 * T * D * (Hq + Hkv)}
    if case["kind"] == "verify":
        n = _drafts(case) + 1
        size, T = {"f16": 2, "bf16": 2, "f32": 4}, int(n.sum())
        read = T * case["V"] * size[case["dtype"]]
        if case["probs"] != "none" and case["temp"] > 0:  # a refused draft's probabilities, about one row in two
            read += case["B"] // 2 * case["V"] * size[case["probs"]]
        return {"bytes": read + 8 * T + 16 * case["B"], "flops": 4 * T * case["V"]}
    kv, new = _lens(case)
    W, S = case["window"], case["sinks"]
    first = np.maximum(kv - new + 1 - W, 0)
    used = int((np.minimum(first, S) + kv - first)[new > 0].sum())
    seen = 0
    for n, L in zip(new, kv):
        last = np.arange(L - n, L)
        low = np.maximum(last + 1 - W, 0)
        seen += int((last + 1 - low + np.minimum(low, S)).sum())
    return {"bytes": used * _row_bytes(case) + 4 * int(new.sum()) * case["Hq"] * case["D"],
            "flops": 4 * case["Hq"] * case["D"] * seen}


# --------------------------------------------------------------------- exact

def _attend_exact(case, seed):
    s = _attend_state(case, seed)
    kv, new = _lens(case)
    G, ps, at = case["Hq"] // case["Hkv"], case["ps"], 0
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        n, L = int(new[b]), int(kv[b])
        if not n:
            continue
        t = torch.arange(L, device="cuda")
        t = t[(t < case["sinks"]) | (t >= L - n + 1 - case["window"])]
        page = s["table"][b, t // ps].long()
        rows = []
        for pool in (s["k"], s["v"]):
            got = [x[page, :, t % ps].double() for x in pool]
            if len(got) == 3:
                got = [got[0] * got[1].repeat_interleave(64, -1) + got[2].repeat_interleave(64, -1)]
            rows.append(got[0])
        me = torch.arange(L - n, L, device="cuda")[:, None]
        hidden = (t > me) | ((t <= me - case["window"]) & (t >= case["sinks"]))
        for h in range(case["Hq"]):
            w = s["q"][at:at + n, h].double() @ rows[0][:, h // G].T * s["scale"]
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h] = w @ rows[1][:, h // G]
        at += n
    return out


def _rope_exact(case, seed):
    s = _rope_state(case, seed)
    D, R = case["D"], case["R"]
    first = torch.arange(R // 2, device="cuda") * (1 if case["pairs"] == "half" else 2)
    second = first + (R // 2 if case["pairs"] == "half" else 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None, None] * s["freqs"])
    got = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        got.append(x)
    q, k = got
    if not case["write"]:
        return dict(q=q, k=k)
    dt, out = DTYPE[case["dtype"]], {"q": q}
    page, off = s["slots"].long() // case["ps"], s["slots"].long() % case["ps"]
    for name, pool, x in (("k", s["pools"][0], k), ("v", s["pools"][1], s["v"].double())):
        if case["q8"]:
            out[name] = None  # (an 8-bit value turns on the roundings before it)
        else:
            out[name] = pool[0].double()
            out[name][page, :, off] = x
    return out


def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers
    return (_attend_exact if case["kind"] == "attend" else _rope_exact)(case, seed)
