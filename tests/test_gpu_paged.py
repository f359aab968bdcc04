"""The paged KV cache's operators on the GPU: plans against plain Python, writes
and reads against the definition, attention against fp64 numpy over each row's
own keys."""
import numpy as np
import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
# half a step of a rounding to the type, relative to the value
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _say(*a):
    print(*a, flush=True)


# ------------------------------------------------------------------- the plan

def _device_plan(seq, new, table, stack, count, page, T, keep):
    from gmlx_amd import ops
    dev = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    tab, st = dev(table), dev(stack)
    args = (dev(seq), dev(new), tab, st, dev([count]), page, T)
    p = ops.paged_plan(*args, keep_lens=None if keep is None else dev(keep))
    got = [p.cu_q, p.kv_lens, p.slots, p.positions, p.free_count, p.refused, tab, st]
    got = [x.cpu().numpy() for x in got]
    again = ops.paged_plan(*args, keep_lens=None if keep is None else dev(keep))
    for a, b in zip(got, [*again[:4], again.free_count, again.refused, tab, st]):
        assert np.array_equal(a, b.cpu().numpy())  # the same call again gives the same
    return got


def _check_plan(seq, new, table, stack, count, page, T, keep=None):
    got = _device_plan(seq, new, table, stack, count, page, T, keep)
    want = ref.plan(seq, new, np.asarray(table), stack, count, page, T, keep)
    names = ("cu_q", "kv_lens", "slots", "positions", "free_count", "refused", "table", "stack")
    for name, a, b in zip(names, got, want):
        assert np.array_equal(a.reshape(-1), np.asarray(b).reshape(-1)), name
    return got


def _rows(rng, B, page, width, used, spare):
    """Rows of `used` tokens with their pages, and a free stack of the spare ones."""
    have = [-(-u // page) for u in used]
    n_pages = sum(have) + spare
    order = rng.permutation(n_pages)
    table, at = np.full((B, width), -7, np.int32), 0
    for b, h in enumerate(have):
        table[b, :h] = order[at:at + h]
        at += h
    stack = np.full(n_pages, -9, np.int32)
    stack[:spare] = order[at:]
    return table, stack, spare


@pytest.mark.parametrize("B,page,hi,n", [(1, 16, 1, 1), (1, 16, 500, 4000), (3, 64, 300, 1), (8, 16, 4000, 5),
                                         (65, 32, 900, 40), (300, 128, 9000, 3), (1025, 16, 200, 2),
                                         (2048, 16, 100, 17)])
def test_plan(B, page, hi, n):
    rng = np.random.default_rng(B * page + n)
    seq = rng.integers(0, hi + 1, B)
    new = rng.integers(0, n + 1, B)
    keep = np.where(rng.random(B) < 0.4, rng.integers(0, hi + 1, B), seq)  # (past seq: all of it)
    keep[rng.random(B) < 0.1] = 0
    width = (hi + n) // page + 2
    table, stack, count = _rows(rng, B, page, width, seq, B * (n // page + 2))
    T = int(new.sum()) + 5
    _say("plan", B, page, hi, n, T)
    _check_plan(seq, new, table, stack, count, page, T, keep)
    _check_plan(seq, new, table, stack, count, page, T)
    _check_plan(seq, new, table, stack, count, page, max(0, T - 9), keep)  # fewer slots than tokens
    # a stack that runs out at some row, at once, and one that is just long enough
    base = np.minimum(keep, seq)
    need = np.maximum(-(-(base + new) // page) - -(-seq // page), 0).sum()
    give = np.maximum(-(-seq // page) - -(-(base + new) // page), 0).sum()
    for c in {0, max(0, int(need - give)), max(0, int(need - give) - 1), count // 7}:
        _check_plan(seq, new, table, stack, c, page, T, keep)


def test_plan_refuses_a_row_that_the_table_cannot_hold():
    rng = np.random.default_rng(3)
    table, stack, count = _rows(rng, 4, 16, 3, [40, 48, 0, 16], 9)
    got = _check_plan([40, 48, 0, 16], [8, 1, 49, 20], table, stack, count, 16, 80)
    assert got[5].tolist() == [0, 1, 1, 0]
    # lengths that no state has: negative ones count as 0, past the table as its width
    _check_plan([-5, 1000, 3, 7], [-1, 0, 2, 1], np.abs(table), stack, count, 16, 8, [0, 999, -4, 7])


def test_plan_of_lengths_that_pass_31_bits_together():
    """Rows too long for the table are refused, the free pages stay, and nothing
    outside the tables is read or written."""
    rng = np.random.default_rng(5)
    table, stack, count = _rows(rng, 4, 16, 3, [16, 20, 0, 5], 6)
    big = 2 ** 31 - 1
    got = _device_plan([16, 20, 0, 5], [big, big, big, big], table, stack, count, 16, 3000, None)
    assert got[5].tolist() == [1, 1, 1, 1] and got[4].tolist() == [6] and (got[2] == -1).all()
    assert np.array_equal(got[6], table) and np.array_equal(got[7], stack)
    got = _device_plan([16, 20, 0, 5], [big, big, 3, 3], table, stack, count, 16, 3000, None)
    assert got[5].tolist() == [1, 1, 0, 0] and ((got[2] >= -1) & (got[2] < 16 * len(stack))).all()


def test_plan_ends_requests_and_reuses_their_pages():
    rng = np.random.default_rng(4)
    seq = [100, 33, 17, 64]
    table, stack, count = _rows(rng, 4, 16, 9, seq, 0)
    # nothing free: row 1's and row 2's pages go back and rows 0 and 3 take them
    got = _check_plan(seq, [16, 0, 0, 20], table, stack, count, 16, 36, [100, 0, 0, 64])
    assert got[5].tolist() == [0, 0, 0, 0] and got[4].tolist() == [2]


# -------------------------------------------------------------- write and read

def _bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _pool(shape, dt, q8, layout, fill=None):
    """k, v (and their scales and biases) [n_pages, Hkv, page, D] in a memory
    layout: 'head' as shaped, 'token' [n_pages, page, Hkv, D] permuted, 'mixed'
    K and V of a page side by side."""
    n, H, P, D = shape

    def make(D, dtype):
        if layout == "token":
            ts = [torch.zeros(n, P, H, D, dtype=dtype, device="cuda").permute(0, 2, 1, 3) for _ in range(2)]
        elif layout == "mixed":
            both = torch.zeros(n, 2, H, P, D, dtype=dtype, device="cuda")
            ts = [both[:, 0], both[:, 1]]
        else:
            ts = [torch.zeros(n, H, P, D, dtype=dtype, device="cuda") for _ in range(2)]
        if fill is not None:
            for t in ts:
                t.fill_(fill if dtype != torch.uint8 else 255)
        return ts
    if not q8:
        return make(D, dt), {}
    (ks, vs), (kb, vb) = make(D // 64, dt), make(D // 64, dt)
    return make(D, torch.uint8), dict(k_scales=ks, k_biases=kb, v_scales=vs, v_biases=vb)


def _quantised(x, dt):
    """(q, scale, bias) of rows [..., D] by the definition, in fp64 but for the
    16-bit rounding of the scale."""
    g = x.double().cpu().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 255).to(dt).double()
    q = torch.where(s[..., None] == 0, 0.0, ((g - lo[..., None]) / s[..., None]).round().clamp(0, 255))
    return q.flatten(-2).to(torch.uint8), s.to(dt), lo.to(dt)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D,H,P,T,layout", [(64, 1, 16, 1, "head"), (96, 3, 32, 37, "token"), (128, 8, 16, 33, "mixed"),
                                            (256, 2, 64, 100, "head"), (512, 1, 128, 9, "token")])
def test_write_and_read_16bit(dt, D, H, P, T, layout):
    from gmlx_amd import ops
    torch.manual_seed(D + T)
    n = T // P + 3
    (k, v), _ = _pool((n, H, P, D), dt, False, layout, fill=3.0)
    # rows from a packed q|k|v block: strides of their own
    rows = torch.randn(T, 3 * H, D, device="cuda").to(dt)
    x, y = rows[:, H:2 * H], rows[:, 2 * H:]
    slots = torch.randperm(n * P, device="cuda")[:T].int()
    if T > 4:
        slots[1], slots[3], slots[4] = -1, n * P, 2 ** 31 - 1  # no slots of the pool
    _say("write16", dt, D, H, P, T, layout)
    before = k.clone(), v.clone()
    ops.paged_write(x, y, k, v, slots)
    ok = (slots >= 0) & (slots < n * P)
    s = slots[ok].long()
    for pool, old, new in ((k, before[0], x), (v, before[1], y)):
        old[s // P, :, s % P] = new[ok]
        assert np.array_equal(_bits(pool), _bits(old))
    got = ops.paged_read(k, v, slots)
    for g, new in zip(got, (x, y)):
        assert np.array_equal(_bits(g), _bits(torch.where(ok[:, None, None], new, 0)))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D,H,P,T,layout", [(64, 1, 16, 1, "head"), (128, 8, 16, 33, "head"), (256, 2, 64, 100, "mixed"),
                                            (512, 1, 128, 9, "head")])
def test_write_and_read_8bit(dt, D, H, P, T, layout):
    """Scales within one 16-bit step of the definition's (their fp32 quotient
    rounds once before the 16-bit rounding), biases exact, values the nearest
    of the stored scale, and read back as scale * q + bias rounded once."""
    from gmlx_amd import ops
    torch.manual_seed(D + T)
    n = T // P + 2
    (k, v), sc = _pool((n, H, P, D), dt, True, layout)
    x, y = (torch.randn(T, H, D, device="cuda") * 3 + 1).to(dt), torch.randn(T, H, D, device="cuda").to(dt)
    x[0, 0, :64] = 1.5  # a group of one value: scale 0
    if T > 2:
        y[1, 0, :64] *= 1e-6  # a tiny group
        x[2, 0, 5] = 60000.0  # an outlier
    slots = torch.randperm(n * P, device="cuda")[:T].int()
    _say("write8", dt, D, H, P, T, layout)
    ops.paged_write(x, y, k, v, slots, **sc)
    got = ops.paged_read(k, v, slots, **sc)
    s = slots.long()
    for new, q, a, b, back in ((x, k, sc["k_scales"], sc["k_biases"], got[0]), (y, v, sc["v_scales"], sc["v_biases"], got[1])):
        q, a, b = (t[s // P, :, s % P].cpu() for t in (q, a, b))
        _, want_s, want_b = _quantised(new, dt)
        assert torch.equal(b, want_b)
        af, wf = a.double(), want_s.double()
        tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        assert ((af - wf).abs() <= wf * torch.finfo(dt).eps + tiny).all()
        g, af, bf = new.double().cpu().unflatten(-1, (-1, 64)), af[..., None], b.double()[..., None]
        ideal = torch.where(af == 0, 0.0, (g - bf) / af).clamp(0, 255)
        # nearest: half a step, and the fp32 quotient's own rounding (2 roundings of values up to 255)
        assert ((q.unflatten(-1, (-1, 64)).double() - ideal).abs() <= 0.5 + 255 * 2.0 ** -22).all()
        val = (q.unflatten(-1, (-1, 64)).double() * af + bf).flatten(-2)
        # one fp32 rounding, then the 16-bit one
        room = val.abs() * (HALF[dt] + 2.0 ** -23) + tiny
        assert ((back.cpu().double() - val).abs() <= room).all()


@pytest.mark.parametrize("dt", [F16, BF16])
def test_write_8bit_groups_that_are_not_finite(dt):
    """The group reads as NaN, the others as before; none hides one as a number."""
    from gmlx_amd import ops
    (k, v), sc = _pool((2, 2, 16, 128), dt, True, "head")
    x = torch.randn(5, 2, 128, device="cuda").to(dt)
    slots = torch.arange(5, dtype=torch.int32, device="cuda") + 7
    ops.paged_write(x, x, k, v, slots, **sc)
    clean = ops.paged_read(k, v, slots, **sc)[0]
    y = x.clone()
    y[0, 0, 3], y[1, 1, 64], y[2, 0, 127], y[3, 0, 0] = float("nan"), float("inf"), float("-inf"), float("nan")
    y[3, 0, 1:64] = 1.0
    ops.paged_write(y, x, k, v, slots, **sc)
    got = ops.paged_read(k, v, slots, **sc)
    bad = torch.zeros(5, 2, 2, dtype=torch.bool, device="cuda")
    bad[0, 0, 0] = bad[1, 1, 1] = bad[2, 0, 1] = bad[3, 0, 0] = True
    bad = bad.repeat_interleave(64, -1)
    assert torch.isnan(got[0][bad]).all() and torch.equal(got[0][~bad], clean[~bad])
    assert torch.equal(got[1], clean)


# ------------------------------------------------------------------- attention

class Batch:
    """Rows of (new tokens, keys) over a pool whose other places hold NaN (8-bit:
    NaN scales), with block tables that end in no pages."""

    def __init__(self, rows, Hq, Hkv, D, P, dt, q8=False, layout="head", seed=0, spread=1.0, pad=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.rows, self.dt, self.scale = rows, dt, D ** -0.5
        have = [-(-kv // P) for _, kv in rows]
        n_pages, width = sum(have) + 3, max(have + [1]) + 2
        (k, v), sc = _pool((n_pages, Hkv, P, D), dt, q8, layout, fill=float("nan"))
        order, at = rng.permutation(n_pages), 0
        table = np.full((len(rows), width), -1, np.int32)
        table[:, 1::2] = 2 ** 31 - 1
        self.k, self.v, self.err = [], [], []
        for b, (n, kv) in enumerate(rows):
            table[b, :have[b]] = order[at:at + have[b]]
            at += have[b]
            t = torch.arange(kv)
            page, off = torch.from_numpy(table[b].astype(np.int64))[t // P].cuda(), (t % P).cuda()
            vals = []
            for pool, which in ((k, "k"), (v, "v")):
                x = (torch.randn(kv, Hkv, D, generator=gen) * spread).to(dt)
                if q8:
                    q, s, bi = _quantised(x, dt)
                    pool[page, :, off] = q.cuda()
                    sc[which + "_scales"][page, :, off] = s.cuda()
                    sc[which + "_biases"][page, :, off] = bi.cuda()
                    s, bi = (a.double()[..., None] for a in (s, bi))
                    centred = (q.unflatten(-1, (-1, 64)).double() - 128) * s
                    # 32-bit dequantisation by sums: s (q . k) + b (sum of q)
                    vals += [(centred + 128 * s + bi).flatten(-2).transpose(0, 1).numpy(),
                             centred.abs().flatten(-2).transpose(0, 1).numpy()]
                else:
                    pool[page, :, off] = x.cuda()
                    vals += [x.double().transpose(0, 1).numpy(), x.double().abs().transpose(0, 1).numpy()]
            self.k.append(vals[0])
            self.v.append(vals[2])
            self.err.append(vals[3])
        T = sum(n for n, _ in rows)
        self.q = torch.randn(T + pad, Hq, D, generator=gen).to(dt)
        self.T = T
        self.pool, self.scales = (k, v), sc
        ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.kv_lens = ints(table), ints([kv for _, kv in rows])
        self.cu = np.concatenate([[0], np.cumsum([n for n, _ in rows])])
        self.cu_q = ints(self.cu)

    def run(self, **kw):
        from gmlx_amd import ops
        q = kw.pop("q", self.q.cuda())
        return ops.sdpa_paged(q, *self.pool, self.table, self.kv_lens, self.cu_q, self.scale, **self.scales, **kw)

    def check(self, out):
        """Every element within: the output's rounding, the probabilities' (of
        the values, or of the centred 8-bit ones that they multiply), and the
        32-bit work of scores of up to 2^6 and sums over the keys."""
        u = HALF[self.dt]
        got = out.double().cpu().numpy()
        for b, (n, kv) in enumerate(self.rows):
            if not n:
                continue
            q = self.q[self.cu[b]:self.cu[b + 1]].double().numpy()
            want, far = ref.attention(q, self.k[b], self.v[b], n, self.scale, self.err[b])
            _, mean = ref.attention(q, self.k[b], self.v[b], n, self.scale)
            smax = 1.5 * self.scale * np.abs(q).sum(-1).max() * max(1.0, np.abs(self.k[b]).max() if kv else 1.0)
            # a score's products and sums (D + 4 roundings), the power's argument and value, the sums over kv keys
            f32 = 2.0 ** -24 * (2 * (q.shape[-1] + 8) * smax + 2 * kv + 16)
            room = u * np.abs(want) + u * (1 + u) * far + f32 * (mean + far) + 1e-7
            d = np.abs(got[self.cu[b]:self.cu[b + 1]] - want)
            assert np.isfinite(d).all() and (d <= room).all(), (b, n, kv, (d / room).max())


SHAPES = [(128, 32, 8), (64, 8, 8), (96, 12, 3), (256, 16, 2), (128, 5, 1), (512, 8, 1), (64, 64, 2), (128, 48, 1)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D,Hq,Hkv", SHAPES)
def test_attention_shapes(D, Hq, Hkv, dt):
    rows = [(1, 1), (1, 15), (0, 40), (1, 16), (1, 33), (3, 3), (7, 7 + 64), (0, 0), (5, 2), (2, 0), (1, 700),
            (40, 333), (1, 0)]
    _say("attend", D, Hq, Hkv, dt)
    b = Batch(rows, Hq, Hkv, D, 16, dt, seed=D + Hq)
    b.check(b.run())


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D,Hq,Hkv", [s for s in SHAPES if s[0] != 96])
def test_attention_8bit(D, Hq, Hkv, dt):
    rows = [(1, 1), (1, 15), (0, 40), (1, 32), (3, 3), (7, 7 + 64), (5, 2), (2, 0), (1, 700), (40, 333)]
    _say("attend8", D, Hq, Hkv, dt)
    b = Batch(rows, Hq, Hkv, D, 32, dt, q8=True, seed=D + Hq)
    b.check(b.run())


@pytest.mark.parametrize("q8,layout", [(False, "token"), (False, "mixed"), (True, "mixed")])
@pytest.mark.parametrize("P", [16, 64, 256, 1024])
def test_attention_pages_and_layouts(P, q8, layout):
    rows = [(1, P), (1, P + 1), (1, 2 * P - 1), (9, 2 * P + 5), (1, 1500), (70, 1200)]
    _say("pages", P, q8, layout)
    b = Batch(rows, 16, 2, 128, P, F16, q8=q8, layout=layout, seed=P)
    b.check(b.run())


@pytest.mark.parametrize("n,kv", [(1, 9000), (2, 5000), (16, 3100), (65, 2049), (129, 129), (300, 2500), (513, 1030)])
@pytest.mark.parametrize("dt,q8", [(F16, False), (BF16, False), (BF16, True)])
def test_attention_chunks(n, kv, dt, q8):
    _say("chunk", n, kv, dt, q8)
    b = Batch([(n, kv), (1, 77), (n // 2, kv // 3 + n)], 8, 2, 128, 64, dt, q8=q8, seed=n)
    b.check(b.run())


def test_attention_large_scores():
    """Scores far apart: probabilities from 1 down to 2^-100 and below."""
    for dt in (F16, BF16):
        _say("large", dt)
        b = Batch([(1, 600), (33, 400)], 8, 2, 64, 16, dt, seed=5, spread=5.0)
        b.check(b.run())


@pytest.mark.parametrize("D,Hq,Hkv,q8", [(128, 32, 8, False), (128, 32, 8, True), (256, 16, 2, False), (64, 8, 8, False)])
def test_row_equals_the_call_on_the_row_alone(D, Hq, Hkv, q8):
    """Bit for bit, and the same at every call."""
    from gmlx_amd import ops
    rows = [(1, 5000), (1, 130), (200, 1700), (4, 2600), (1, 1), (37, 37)]
    b = Batch(rows, Hq, Hkv, D, 16, BF16, q8=q8, seed=9)
    full = b.run()
    assert torch.equal(full, b.run())
    for i, (n, kv) in enumerate(rows):
        lo, hi = int(b.cu[i]), int(b.cu[i + 1])
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        _say("alone", D, q8, n, kv)
        one = ops.sdpa_paged(b.q[lo:hi].cuda(), *b.pool, b.table[i:i + 1], b.kv_lens[i:i + 1], cu, b.scale, max_q=n,
                             max_kv=kv, **b.scales)
        assert torch.equal(one, full[lo:hi]), (n, kv)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,kv,Hq", [(5, 70, 8), (40, 90, 8), (150, 400, 8), (150, 400, 32)])
def test_values_that_a_token_does_not_see(n, kv, Hq, dt):
    """Infinities and NaN in the keys and values of later tokens leave earlier
    ones as they are; the tokens that see them get what the sum gives."""
    base = Batch([(n, kv), (1, 20)], Hq, 2, 128, 16, dt, seed=n)
    clean = base.run()
    k, v = base.pool
    P = 16
    hit = kv - n // 2 - 1          # a key in the middle of the chunk
    page, off = int(base.table[0, hit // P]), hit % P
    for bad, what in ((float("inf"), "v"), (float("-inf"), "v"), (float("nan"), "v"), (float("nan"), "k"),
                      (float("inf"), "k")):
        _say("hidden", bad, what, n, kv, dt)
        pool = (v if what == "v" else k)
        was = pool[page, :, off].clone()
        pool[page, 1, off, 3] = bad
        out = base.run()
        pool[page, :, off] = was
        first = hit - (kv - n)     # the first new token that sees it
        half = Hq // 2
        assert torch.equal(out[:first], clean[:first]) and torch.equal(out[n:], clean[n:])
        assert torch.equal(out[:, :half], clean[:, :half])  # the other kv head
        seen = out[first:n, half:]
        if what == "v":
            col = seen[:, :, 3].float()
            # (a probability that rounds to 0 makes 0 * inf, so NaN is possible beside the infinity)
            assert (torch.isnan(col).all() if bad != bad else (torch.isnan(col) | (col == bad)).all())
            rest = [d for d in range(128) if d != 3]
            assert torch.equal(seen[:, :, rest], clean[first:n, half:][:, :, rest])
        elif bad != bad:
            assert torch.isnan(seen).all()


def test_hidden_scales_of_an_8bit_pool():
    base = Batch([(40, 90), (1, 20)], 8, 2, 128, 16, F16, q8=True, seed=2)
    clean = base.run()
    hit, P = 70, 16
    page, off, first = int(base.table[0, hit // P]), hit % P, 70 - 50
    for name in ("v_scales", "v_biases", "k_scales"):
        t = base.scales[name]
        was = t[page, 1, off, 1].clone()
        t[page, 1, off, 1] = float("nan")
        out = base.run()
        t[page, 1, off, 1] = was
        _say("hidden scale", name)
        assert torch.equal(out[:first], clean[:first]) and torch.equal(out[:, :4], clean[:, :4])
        assert torch.isnan(out[first:40, 4:, 64:]).all()


def test_pages_outside_the_pool_are_not_seen():
    """Keys of a table entry that is no page of the pool are left out."""
    from gmlx_amd import ops
    for n, kv, bad in ((1, 200, -1), (1, 200, 10 ** 6), (30, 200, -1), (30, 200, 2 ** 31 - 1)):
        b = Batch([(n, kv)], 8, 2, 128, 32, F16, seed=7)
        tab = b.table.clone()
        tab[0, 2] = bad
        _say("bad page", n, kv, bad)
        out = ops.sdpa_paged(b.q.cuda(), *b.pool, tab, b.kv_lens, b.cu_q, b.scale)
        keep = [t for t in range(kv) if t // 32 != 2]
        for i in range(n):
            vis = [t for t in keep if t <= kv - n + i]
            want, far = ref.attention(b.q[i:i + 1].double().numpy(), b.k[0][:, vis], b.v[0][:, vis], 1, b.scale)
            d = np.abs(out[i:i + 1].double().cpu().numpy() - want)
            assert (d <= HALF[F16] * (np.abs(want) + far) + 1e-4 * far).all()


def test_rows_behind_the_last_sequence_and_strides():
    """A padded batch into a given output; q a slice of a packed q|k|v block."""
    for q8 in (False, True):
        b = Batch([(1, 300), (20, 150), (0, 5)], 8, 2, 128, 16, BF16, q8=q8, seed=3, pad=11)
        out = torch.full((32, 8, 128), 7.0, dtype=BF16, device="cuda")
        packed = torch.full((32, 12 * 128), float("nan"), dtype=BF16, device="cuda")
        packed[:21, :8 * 128] = b.q[:21].reshape(21, -1).cuda()
        got = b.run(q=packed[:, :8 * 128].unflatten(1, (8, 128)), out=out)
        assert got.data_ptr() == out.data_ptr() and (out[21:] == 7.0).all()
        b.check(out[:21])
        assert torch.equal(out[:21], b.run()[:21])
        wide = torch.zeros(32, 16, 128, dtype=BF16, device="cuda")
        b.run(out=wide[:, 3:11])
        assert torch.equal(wide[:21, 3:11], out[:21]) and (wide[:, :3] == 0).all() and (wide[:, 11:] == 0).all()


def test_bounds_cut_longer_rows():
    """max_q and max_kv below the rows' lengths: the first max_q tokens are
    computed, over the first max_kv keys."""
    b = Batch([(6, 100), (2, 50)], 8, 2, 128, 16, F16, seed=3)
    out = torch.full((8, 8, 128), 7.0, dtype=F16, device="cuda")
    b.run(out=out, max_q=4)
    full = b.run()
    assert (out[4:6] == 7.0).all() and torch.equal(out[6:], full[6:])
    # (four tokens may take another kernel than six: the same sums in another order)
    cut = full.clone()
    cut[:4] = out[:4]
    b.check(cut)
    b.run(out=out, max_kv=64)
    assert torch.equal(out[6:], full[6:])
    assert torch.isfinite(out).all()
    # malformed tables: lengths past the table, a cu_q that runs backwards or past T
    b.kv_lens = torch.tensor([10 ** 9, -3], dtype=torch.int32, device="cuda")
    b.cu_q = torch.tensor([4, 2, 90], dtype=torch.int32, device="cuda")
    b.run(out=out)
    torch.cuda.synchronize()


def test_large_pool_offsets():
    """Pages that start past 2^31 and 2^32 bytes and elements of the pool."""
    from gmlx_amd import ops
    P, H, D = 64, 4, 128
    n = (5 << 30) // (2 * P * H * D)  # 5 GiB of K, 2.7 G elements
    dt = F16
    k, v = (torch.zeros(n, H, P, D, dtype=dt, device="cuda") for _ in range(2))
    pages = [n - 1, 1, n // 2 + 3, n - 2, (1 << 31) // (P * H * D) + 1]
    kv = 5 * P - 7
    x, y = (torch.randn(kv, H, D, device="cuda").to(dt) for _ in range(2))
    slots = torch.tensor([pages[t // P] * P + t % P for t in range(kv)], dtype=torch.int32, device="cuda")
    ops.paged_write(x, y, k, v, slots)
    got = ops.paged_read(k, v, slots)
    assert torch.equal(got[0], x) and torch.equal(got[1], y)
    table = torch.tensor([pages], dtype=torch.int32, device="cuda")
    for m in (1, 33):
        q = torch.randn(m, 8, D, device="cuda").to(dt)
        cu = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        _say("large pool", m)
        out = ops.sdpa_paged(q, k, v, table, torch.tensor([kv], dtype=torch.int32, device="cuda"), cu, D ** -0.5)
        want, far = ref.attention(q.double().cpu().numpy(), x.double().cpu().numpy().transpose(1, 0, 2),
                                  y.double().cpu().numpy().transpose(1, 0, 2), m, D ** -0.5)
        d = np.abs(out.double().cpu().numpy() - want)
        assert (d <= HALF[dt] * (np.abs(want) + far) + 1e-4 * far).all()


# --------------------------------------------------------- the operators together

class Serving:
    """A pool, its tables and a step over them: plan, write, attend."""

    def __init__(self, B, Hq, Hkv, D, P, n_pages, width, dt, q8):
        from gmlx_amd import ops
        self.ops, self.dt, self.P, self.Hq, self.Hkv, self.D = ops, dt, P, Hq, Hkv, D
        self.scale = D ** -0.5
        (self.k, self.v), self.sc = _pool((n_pages, Hkv, P, D), dt, q8, "mixed", fill=float("nan"))
        i32 = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((B, width), -1, **i32)
        self.free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(B)).to(**i32)
        self.count = torch.tensor([n_pages], **i32)
        self.seq = torch.zeros(B, **i32)

    def step(self, new, keep, q, k, v, max_q, out=None):
        """In place of the state, as a captured graph has it."""
        ops = self.ops
        p = ops.paged_plan(self.seq, new, self.table, self.free, self.count, self.P, q.shape[0], keep_lens=keep)
        self.seq.copy_(p.kv_lens)
        self.count.copy_(p.free_count)
        ops.paged_write(k, v, self.k, self.v, p.slots, **self.sc)
        out = ops.sdpa_paged(q, self.k, self.v, self.table, p.kv_lens, p.cu_q, self.scale, max_q=max_q, out=out, **self.sc)
        return p, out

    def state(self):
        return [self.table, self.free, self.count, self.seq, self.k, self.v, *self.sc.values()]

    def row(self, b):
        """The row's cached K and V in fp64 (Hkv, kv, D), and what a probability's
        rounding multiplies: |V|, of an 8-bit pool the centred values'."""
        kv = int(self.seq[b])
        t = torch.arange(kv, device="cuda")
        page, off = self.table[b].long()[t // self.P], t % self.P
        vals = []
        for pool, x in ((self.k, "k"), (self.v, "v")):
            z = pool[page, :, off].double()
            far = z.abs()
            if self.sc:
                s, bi = (self.sc[x + name][page, :, off].double().repeat_interleave(64, -1) for name in ("_scales", "_biases"))
                z, far = z * s + bi, ((z - 128) * s).abs()
            vals += [z, far]
        return [x.transpose(0, 1).cpu().numpy() for x in (vals[0], vals[2], vals[3])]

    def check(self, q, out, b, lo, n):
        k, v, err = self.row(b)
        kv = k.shape[1]
        x = q[lo:lo + n].double().cpu().numpy()
        want, far = ref.attention(x, k, v, n, self.scale, err)
        _, mean = ref.attention(x, k, v, n, self.scale)
        u = HALF[self.dt]
        smax = 1.5 * self.scale * np.abs(x).sum(-1).max() * max(1.0, np.abs(k).max())
        f32 = 2.0 ** -24 * (2 * (x.shape[-1] + 8) * smax + 2 * kv + 16)  # (as Batch.check counts)
        room = u * np.abs(want) + u * (1 + u) * far + f32 * (mean + far) + 1e-7
        d = np.abs(out[lo:lo + n].double().cpu().numpy() - want)
        assert np.isfinite(d).all() and (d <= room).all(), (b, n, kv, (d / room).max())


# (new tokens, tokens kept) of four rows a step: prompts, decoding, drafts of
# which some are rejected, an ended request whose row and pages go to the next
# one, a row that the pool has no pages for
STEPS = [([70, 0, 5, 33], None), ([1, 40, 1, 1], None), ([1, 1, 1, 1], None), ([5, 5, 5, 5], None),
         ([5, 1, 5, 2], [74, 46, 10, 37]), ([130, 1, 0, 1], [0, 47, 14, 39]), ([1, 1, 1, 1000], None),
         ([1, 1, 1, 1], [130, 47, 14, 0]), ([0, 0, 0, 17], None)]


def _inputs(s, T, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda h: torch.randn(T, h, s.D, device="cuda", generator=gen).to(s.dt)  # noqa: E731
    return new(s.Hq), new(s.Hkv), new(s.Hkv)


@pytest.mark.parametrize("dt,q8,Hq,Hkv,D", [(BF16, False, 8, 2, 128), (F16, True, 8, 2, 128), (F16, False, 4, 4, 64),
                                           (BF16, True, 16, 2, 256)])
def test_steps_of_a_serving_loop(dt, q8, Hq, Hkv, D):
    s = Serving(4, Hq, Hkv, D, 16, 40, 70, dt, q8)
    i32 = dict(dtype=torch.int32, device="cuda")
    model = [torch.zeros(0, Hkv, D, dtype=dt, device="cuda") for _ in range(4)]  # keys in order
    for i, (new, keep) in enumerate(STEPS):
        T = sum(new) + 3  # (padded)
        q, k, v = _inputs(s, T, i)
        _say("step", i, dt, q8, D, new, keep)
        p, out = s.step(torch.tensor(new, **i32), None if keep is None else torch.tensor(keep, **i32), q, k, v, max(new))
        refused, lo = p.refused.tolist(), 0
        assert refused == [0, 0, 0, int(new[3] == 1000)]
        for b, n in enumerate(new):
            if not refused[b]:
                kept = model[b] if keep is None else model[b][:keep[b]]
                model[b] = torch.cat([kept, k[lo:lo + n]])
                if not q8:
                    assert np.array_equal(s.row(b)[0], model[b].double().transpose(0, 1).cpu().numpy())
                if n:
                    s.check(q, out, b, lo, n)
            assert int(s.seq[b]) == len(model[b])
            lo += n
        pages = [int(x) for b in range(4) for x in s.table[b, :-(-len(model[b]) // 16)]]
        pages += s.free[:int(s.count)].tolist()
        assert sorted(pages) == list(range(40))  # every page once


@pytest.mark.parametrize("q8", [False, True])
def test_step_captured_and_replayed(q8):
    """A step of two new tokens a row, of which the next keeps one or both, in a
    graph that updates the state in place; eager work between the replays; every
    replay bit for bit as the eager step."""
    B, i32 = 6, dict(dtype=torch.int32, device="cuda")

    def fresh():
        s = Serving(B, 8, 2, 128, 16, 200, 40, BF16, q8)
        q, k, v = _inputs(s, 6 * 90, 99)
        s.step(torch.tensor([90, 1, 33, 500 - 300, 16, 2], **i32), None, q, k, v, 200)
        return s
    eager, live = fresh(), fresh()
    T = 2 * B
    new = torch.full((B,), 2, **i32)
    hold = [*_inputs(live, T, 0), torch.zeros(B, **i32)]
    hold[3].copy_(live.seq)
    outs = torch.zeros(T, 8, 128, dtype=BF16, device="cuda")
    saved = [x.clone() for x in live.state()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (builds what the first call builds, on another stream than the tensors')
        live.step(new, hold[3], *hold[:3], 2, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(live.state(), saved):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        live.step(new, hold[3], *hold[:3], 2, out=outs)
    for x, y in zip(live.state(), saved):
        x.copy_(y)
    for i in range(7):
        q, k, v = _inputs(live, T, 100 + i)
        keep = eager.seq - torch.tensor([(i + b) % 2 if i else 0 for b in range(B)], **i32)
        for x, y in zip(hold, (q, k, v, keep)):
            x.copy_(y)
        _say("replay", i, q8)
        graph.replay()
        _, want = eager.step(new, keep, q, k, v, 2)
        torch.cuda.synchronize()
        assert torch.equal(outs, want)
        for x, y in zip(live.state(), eager.state()):
            assert np.array_equal(_bits(x), _bits(y))


def test_two_graphs_replayed_at_once():
    """Each call of a graph has a workspace of its own: two graphs captured one
    after the other, replayed on two streams, beside eager calls on a third."""
    from gmlx_amd import ops
    batches = [Batch([(1, 6000), (1, 3000), (1, 9000)], 8, 2, 128, 16, F16, seed=1),
               Batch([(1, 8000), (1, 7000)], 8, 2, 128, 16, F16, seed=2)]
    want = [b.run() for b in batches]
    qs = [b.q.cuda() for b in batches]
    graphs, outs = [], []
    for b, q in zip(batches, qs):
        g, out = torch.cuda.CUDAGraph(), torch.zeros_like(q)
        with torch.cuda.graph(g):
            for _ in range(20):
                ops.sdpa_paged(q, *b.pool, b.table, b.kv_lens, b.cu_q, b.scale, out=out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(4):
        for out in outs:
            out.zero_()
        _say("two graphs", i)
        for st, g in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        more = [b.run() for b in batches for _ in range(5)]
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
        for j, m in enumerate(more):
            assert torch.equal(m, want[j // 5])


def test_ops_refuse_what_they_cannot_take():
    """By an error, before any launch."""
    from gmlx_amd import ops
    b = Batch([(1, 40), (2, 20)], 8, 2, 128, 16, F16, seed=1)
    e = Batch([(1, 40), (2, 20)], 8, 2, 128, 16, F16, q8=True, seed=1)
    (k, v), q = b.pool, b.q.cuda()
    x = torch.zeros(3, 2, 128, dtype=F16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")

    def attend(**kw):
        a = dict(q=q, k_cache=k, v_cache=v, block_table=b.table, kv_lens=b.kv_lens, cu_q=b.cu_q, scale=1.0)
        ops.sdpa_paged(**{**a, **kw})
    with_scales = dict(k_cache=e.pool[0], v_cache=e.pool[1], **e.scales)
    for bad in (dict(q=q.bfloat16()), dict(q=q[:, :3]), dict(q=q[0]), dict(q=q[..., :64]), dict(q=q.cpu()),
                dict(k_cache=k[:, :, :, :64]), dict(v_cache=v[:2]), dict(k_cache=k.bfloat16()),
                dict(k_cache=k.float(), v_cache=v.float()), dict(k_cache=k.transpose(2, 3), v_cache=v.transpose(2, 3)),
                dict(block_table=b.table.long()), dict(block_table=b.table[:1]), dict(block_table=b.table.cpu()),
                dict(kv_lens=b.kv_lens.long()), dict(cu_q=b.cu_q[:2]), dict(max_q=0), dict(max_kv=-1), dict(max_kv=0),
                dict(out=torch.empty(3, 8, 128, device="cuda")), dict(out=torch.empty(4, 8, 128, dtype=F16, device="cuda")),
                dict(out=torch.empty(3, 128, 8, dtype=F16, device="cuda").transpose(1, 2)),
                dict(k_cache=e.pool[0], v_cache=e.pool[1]), {**with_scales, "v_biases": None},
                {**with_scales, "k_scales": e.scales["k_scales"].bfloat16()},
                {**with_scales, "k_scales": e.scales["k_scales"][:2]}, {**with_scales, "k_cache": k, "v_cache": v}):
        with pytest.raises((ValueError, RuntimeError)):
            attend(**bad)
    for bad in (dict(k=x.float()), dict(k=x[:2]), dict(v=x[:, :1]), dict(slots=slots.long()), dict(slots=slots[:2]),
                dict(v_cache=v.bfloat16())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_write(**{**dict(k=x, v=x, k_cache=k, v_cache=v, slots=slots), **bad})
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    plan = dict(seq_lens=one, new_lens=one, block_table=b.table, free_pages=slots, free_count=one[:1], page_size=16,
                max_tokens=2)
    for bad in (dict(new_lens=one[:1]), dict(page_size=24), dict(page_size=8), dict(max_tokens=-1),
                dict(free_count=one), dict(keep_lens=one.long()), dict(block_table=b.table[:1]),
                dict(seq_lens=torch.ones(3000, dtype=torch.int32, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_plan(**{**plan, **bad})
    attend()


def test_calls_without_tokens_or_keys():
    from gmlx_amd import ops
    b = Batch([(0, 40), (0, 0)], 8, 2, 128, 16, F16, seed=1)
    assert b.run().shape == (0, 8, 128)
    x = torch.zeros(0, 2, 128, dtype=F16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    ops.paged_write(x, x, *b.pool, none)
    assert ops.paged_read(*b.pool, none)[0].shape == (0, 2, 128)
    out = torch.full((3, 8, 128), 7.0, dtype=F16, device="cuda")  # all rows padding
    b.run(q=torch.ones_like(out), out=out)
    assert (out == 7.0).all()


@pytest.mark.parametrize("q8", [False, True])
def test_many_rows(q8):
    """More rows than a wave scans at once, chunks among them, in a workspace
    whose slots follow one another."""
    rng = np.random.default_rng(8)
    rows = [(1, int(kv)) for kv in rng.integers(1, 900, 140)]
    for i in range(10):
        rows.insert(int(rng.integers(0, len(rows))), (int(rng.integers(2, 120)), int(rng.integers(400, 900))))
    rows[70:70] = [(0, 30), (0, 0), (3, 1)]
    _say("many rows", len(rows), q8)
    b = Batch(rows, 8, 2, 64, 32, F16, q8=q8, seed=4)
    out = b.run()
    b.check(out)
    # the longest chunk and a decode row behind it, alone
    longest = max(range(len(rows)), key=lambda r: rows[r][0])
    for r in (longest, len(rows) - 1):
        lo, hi = int(b.cu[r]), int(b.cu[r + 1])
        from gmlx_amd import ops
        one = ops.sdpa_paged(b.q[lo:hi].cuda(), *b.pool, b.table[r:r + 1], b.kv_lens[r:r + 1],
                             torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"), b.scale, **b.scales)
        assert torch.equal(one, out[lo:hi])


@pytest.mark.parametrize("D,Hq,q8", [(64, 2, False), (128, 4, True), (256, 1, False)])
def test_long_prompt(D, Hq, q8):
    """A prompt of 4100 tokens and one of 3000 behind 2000: sampled tokens."""
    rows = [(4100, 4100), (3000, 5000)]
    b = Batch(rows, Hq, 1, D, 64, BF16, q8=q8, seed=D)
    _say("long prompt", D, Hq, q8)
    out = b.run().double().cpu().numpy()
    u, rng = HALF[BF16], np.random.default_rng(D)
    for r, (n, kv) in enumerate(rows):
        for i in [0, 1, n - 1, *rng.integers(0, n, 12)]:
            t, see = int(b.cu[r]) + int(i), kv - n + int(i) + 1
            q, k, v = b.q[t:t + 1].double().numpy(), b.k[r][:, :see], b.v[r][:, :see]
            want, far = ref.attention(q, k, v, 1, b.scale, b.err[r][:, :see])
            _, mean = ref.attention(q, k, v, 1, b.scale)
            smax = 1.5 * b.scale * np.abs(q).sum(-1).max() * max(1.0, np.abs(k).max())
            f32 = 2.0 ** -24 * (2 * (D + 8) * smax + 2 * see + 16)  # (as Batch.check counts)
            room = u * np.abs(want) + u * (1 + u) * far + f32 * (mean + far) + 1e-7
            assert (np.abs(out[t:t + 1] - want) <= room).all(), (r, i)


def test_rows_that_share_pages():
    """A common prefix in the same pages: every row as with pages of its own."""
    from gmlx_amd import ops
    P, H, D, n = 16, 2, 128, 12
    k, v = (torch.randn(n, H, P, D, device="cuda").to(BF16) for _ in range(2))
    i32 = dict(dtype=torch.int32, device="cuda")
    shared = torch.tensor([[0, 1, 2, 3, 4], [0, 1, 2, 5, 6], [0, 1, 2, 3, 4]], **i32)
    lens, cu = torch.tensor([75, 66, 50], **i32), torch.tensor([0, 1, 21, 22], **i32)
    q = torch.randn(22, 8, D, device="cuda").to(BF16)
    out = ops.sdpa_paged(q, k, v, shared, lens, cu, 0.1)
    own = torch.randperm(15, device="cuda").int().view(3, 5)
    k2, v2 = (torch.zeros(15, H, P, D, dtype=BF16, device="cuda") for _ in range(2))
    k2[own.long()], v2[own.long()] = k[shared.long()], v[shared.long()]
    assert torch.equal(out, ops.sdpa_paged(q, k2, v2, own, lens, cu, 0.1))


def test_output_in_place_of_the_queries():
    b = Batch([(1, 3000), (60, 700), (3, 40)], 8, 2, 128, 16, BF16, seed=6)
    want, q = b.run(), b.q.cuda()
    b.run(q=q, out=q)
    assert torch.equal(q, want)


@pytest.mark.parametrize("D,Hq,Hkv,q8", [(64, 8, 2, False), (96, 6, 3, False), (128, 8, 2, True), (256, 4, 2, False),
                                         (512, 2, 1, False)])
def test_rows_of_many_splits(D, Hq, Hkv, q8, monkeypatch):
    """More splits than a wave's lanes, with direct grids and with a chunk beside
    them, whose grids are not; the bits of the long row are the same."""
    monkeypatch.setenv("GMLX_KQ_SDPA_SPLIT", "64")
    rows = [(1, 9000), (2, 4500), (1, 300), (0, 7)]
    _say("many splits", D, q8)
    a = Batch(rows, Hq, Hkv, D, 32, BF16, q8=q8, seed=D)
    b = Batch(rows + [(60, 900)], Hq, Hkv, D, 32, BF16, q8=q8, seed=D)
    out, more = a.run(), b.run()
    a.check(out)
    b.check(more)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    from gmlx_amd import ops
    one = ops.sdpa_paged(b.q[:1].cuda(), *b.pool, b.table[:1], b.kv_lens[:1], cu, b.scale, **b.scales)
    assert torch.equal(one, more[:1])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("D", [64, 256])
def test_scales_of_zero_and_below(D, q8):
    """A negative scale is the positive one of -q (whose products the matrix cores
    need not round to the opposite of q's: each against fp64); 0 weighs all alike."""
    b = Batch([(1, 700), (3, 90), (70, 500)], 8, 2, D, 32, F16, q8=q8, seed=D)
    q = b.q.cuda()
    b.scale = -b.scale
    out = b.run()
    b.scale, b.q = -b.scale, -b.q
    b.check(out)
    zero = b.run(q=torch.zeros_like(q))
    b.scale = 0.0
    assert torch.equal(b.run(), zero) and torch.isfinite(zero).all()


@pytest.mark.parametrize("D,Hq,Hkv,q8", [(64, 4, 1, False), (128, 4, 2, True), (256, 2, 1, False)])
def test_long_contexts(D, Hq, Hkv, q8):
    """Rows of 40 k to 70 k keys; each row's bits alone with its own bound, too."""
    from gmlx_amd import ops
    rows = [(1, 65535), (1, 65536), (2, 70001), (1, 40000)]
    _say("long contexts", D, q8)
    b = Batch(rows, Hq, Hkv, D, 256, F16, q8=q8, seed=D)
    out = b.run()
    b.check(out)
    for r, (n, kv) in enumerate(rows):
        lo = int(b.cu[r])
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        one = ops.sdpa_paged(b.q[lo:lo + n].cuda(), *b.pool, b.table[r:r + 1], b.kv_lens[r:r + 1], cu, b.scale, max_q=n,
                             max_kv=kv, **b.scales)
        assert torch.equal(one, out[lo:lo + n]), (n, kv)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 8, 2), (256, 8, 2), (512, 4, 1)])
def test_8bit_values_past_the_largest_fp16(D, Hq, Hkv):
    """A group from 0 to 65504 has the scale 257, and its largest value is 65535:
    in K and in V, for a decode row and a chunk over the same pages."""
    from gmlx_amd import ops
    gen, kv, P = torch.Generator(device="cuda").manual_seed(D), 333, 32
    n = -(-kv // P)
    (k, v), sc = _pool((n, Hkv, P, D), F16, True, "head")
    x, y = (torch.rand(kv, Hkv, D, device="cuda", generator=gen) * 60000 for _ in range(2))
    x[:, :, 5::64] = y[::2, :, 5::64] = 65504.0
    x[:, :, 6::64] = y[:, :, 6::64] = 0.0
    ops.paged_write(x.half(), y.half(), k, v, torch.arange(kv, dtype=torch.int32, device="cuda"), **sc)
    vals = []
    for pool, name in ((k, "k"), (v, "v")):
        q, s, bi = (t.transpose(1, 2).reshape(n * P, Hkv, -1)[:kv].double()
                    for t in (pool, sc[name + "_scales"], sc[name + "_biases"]))
        s, bi = s.repeat_interleave(64, -1), bi.repeat_interleave(64, -1)
        # (rounded probabilities multiply the values, or the centred integers times the scale)
        vals += [(s * q + bi).transpose(0, 1).cpu().numpy(),
                 torch.maximum((s * q + bi).abs(), (s * (q - 128)).abs()).transpose(0, 1).cpu().numpy()]
    assert vals[0].max() == vals[2].max() == 65535.0
    for m in (1, 40):
        q = (torch.randn(m, Hq, D, device="cuda", generator=gen) * 1e-4).half()
        i32 = dict(dtype=torch.int32, device="cuda")
        _say("past fp16", D, m)
        out = ops.sdpa_paged(q, k, v, torch.arange(n, **i32)[None], torch.tensor([kv], **i32),
                             torch.tensor([0, m], **i32), D ** -0.5, **sc)
        qd = q.double().cpu().numpy()
        want, far = ref.attention(qd, vals[0], vals[2], m, D ** -0.5, vals[3])
        smax = 1.5 * D ** -0.5 * np.abs(qd).sum(-1).max() * np.abs(vals[0]).max()
        # (as Batch.check counts, and the rounding of a value's second half: 2^-22)
        f32 = 2.0 ** -24 * (2 * (D + 8) * smax + 2 * kv + 16) + 2.0 ** -22
        room = HALF[F16] * np.abs(want) + HALF[F16] * (1 + HALF[F16]) * far + f32 * 2 * far + 1e-7
        d = np.abs(out.double().cpu().numpy() - want)
        assert np.isfinite(d).all() and (d <= room).all(), (m, (d / room).max())


def _check_tokens(b, out, cut, take=None):
    """As Batch.check, token by token, of rows cut to their first `cut` keys (and
    `take` tokens): token i sees keys up to kv - n + i, of those."""
    u, got = HALF[b.dt], out.double().cpu().numpy()
    for r, (n, kv) in enumerate(b.rows):
        for i in range(n if take is None else min(n, take)):
            t, see = int(b.cu[r]) + i, max(0, min(kv - n + i + 1, cut))
            q, k, v = b.q[t:t + 1].double().numpy(), b.k[r][:, :see], b.v[r][:, :see]
            want, far = ref.attention(q, k, v, 1, b.scale, b.err[r][:, :see])
            _, mean = ref.attention(q, k, v, 1, b.scale)
            smax = 1.5 * b.scale * np.abs(q).sum(-1).max() * max(1.0, np.abs(k).max() if see else 1.0)
            f32 = 2.0 ** -24 * (2 * (q.shape[-1] + 8) * smax + 2 * see + 16)
            room = u * np.abs(want) + u * (1 + u) * far + f32 * (mean + far) + 1e-7
            d = np.abs(got[t:t + 1] - want)
            assert np.isfinite(d).all() and (d <= room).all(), (r, n, kv, i, cut, (d / room).max())


@pytest.mark.parametrize("D,Hq,Hkv,q8,dt", [(128, 8, 2, False, F16), (128, 8, 2, True, BF16), (256, 4, 2, False, BF16),
                                            (256, 4, 2, True, F16), (64, 4, 4, True, F16), (96, 6, 2, False, F16),
                                            (512, 2, 1, False, F16)])
def test_cut_rows_keep_their_causal_line(D, Hq, Hkv, q8, dt):
    """max_kv, or a table narrower than a row, leaves keys out and moves nothing:
    fewer keys than new tokens among them."""
    from gmlx_amd import ops
    rows = [(6, 100), (2, 50), (1, 700), (90, 90), (40, 333), (1, 64), (3, 5), (40, 1300)]
    b = Batch(rows, Hq, Hkv, D, 16, dt, q8=q8, seed=D)
    for cut in (1, 17, 64, 200, 1290):
        _say("cut", D, q8, cut)
        _check_tokens(b, b.run(max_kv=cut), cut)
    full = torch.full((b.T, Hq, D), 7.0, dtype=dt, device="cuda")
    b.run(max_kv=48, max_q=5, out=full)
    _check_tokens(b, full, 48, take=5)
    narrow = ops.sdpa_paged(b.q.cuda(), *b.pool, b.table[:, :4].contiguous(), b.kv_lens, b.cu_q, b.scale, **b.scales)
    _check_tokens(b, narrow, 64)


def test_tables_of_more_keys_than_a_row_can_have():
    """The default bound of a table of 2^31 places is the most keys of a row."""
    from gmlx_amd import ops
    i32 = dict(dtype=torch.int32, device="cuda")
    k, v = (torch.randn(3, 1, 1024, 64, device="cuda").half() for _ in range(2))
    table = torch.full((1, 1 << 21), -1, **i32)
    table[0, :3] = torch.tensor([2, 0, 1], **i32)
    q = torch.randn(1, 2, 64, device="cuda").half()
    lens, cu = torch.tensor([2500], **i32), torch.tensor([0, 1], **i32)
    want = ops.sdpa_paged(q, k, v, table[:, :3].contiguous(), lens, cu, 0.125)
    _say("wide table")
    assert torch.equal(ops.sdpa_paged(q, k, v, table, lens, cu, 0.125), want)


def test_calls_keep_no_memory():
    """An eager call's partials go back to torch's allocator with the call: as
    large as asked for, none kept for later calls or other streams."""
    b = Batch([(1, 6000), (1, 3000), (3, 900), (70, 2000)], 8, 2, 128, 16, F16, seed=1)
    want, q = b.run(), b.q.cuda()
    out = torch.zeros_like(q)
    from gmlx_amd import _lib
    need = _lib.lib().kq_sdpa_paged_workspace_bytes(b.T, 4, 8, 2, 128, b.T, 16 * b.table.shape[1], 0)
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            before = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            b.run(q=q, out=out)
            assert torch.cuda.memory_allocated() == before
            assert torch.cuda.max_memory_allocated() - before <= need + (2 << 20)  # (torch's blocks)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_malformed_rows_stay_inside_the_workspace():
    """A cu_q that counts tokens many times over, in a workspace that holds each
    once: rows past its end are left out, and nothing behind it is written."""
    from gmlx_amd import _lib
    L, T, B, Hq, Hkv, D = _lib.lib(), 500, 300, 8, 2, 128
    b = Batch([(1, 3000)], Hq, Hkv, D, 16, F16, seed=1)
    i32 = dict(dtype=torch.int32, device="cuda")
    cu = torch.zeros(B + 1, **i32)
    cu[1::2], cu[2::4] = T, T - 3  # (500 tokens, none, 3, none again and again)
    table = b.table.repeat(B, 1)
    q = torch.randn(T, Hq, D, device="cuda").half()
    out = torch.zeros_like(q)
    need = L.kq_sdpa_paged_workspace_bytes(T, B, Hq, Hkv, D, T, 3000, 0)
    ws = torch.full((need + (64 << 20),), 77, dtype=torch.uint8, device="cuda")
    (k, v), n = b.pool, b.table.shape[1]
    pool = _lib.PagedPool(k=k.data_ptr(), v=v.data_ptr(), page_stride=k.stride(0), head_stride=k.stride(1),
                          token_stride=k.stride(2), n_pages=k.shape[0], page_size=16, Hkv=Hkv, D=D, dtype=_lib.DTYPE_F16)
    _say("malformed rows", need)
    import ctypes
    rc = L.kq_sdpa_paged(q.data_ptr(), Hq * D, ctypes.byref(pool), table.data_ptr(), n, n,
                         torch.full((B,), 3000, **i32).data_ptr(), cu.data_ptr(), T, B, Hq, T, 3000, D ** -0.5, out.data_ptr(),
                         Hq * D, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and (ws[need:] == 77).all()


@pytest.mark.parametrize("D,Hq,Hkv,q8", [(128, 8, 2, False), (128, 8, 2, True), (64, 4, 1, False), (256, 4, 2, False)])
@pytest.mark.parametrize("split", [None, "64"])
def test_values_of_far_smaller_keys(D, Hq, Hkv, q8, split, monkeypatch):
    """A NaN among the values that a token sees is in its output, though the whole
    split's probabilities round to 0 beside another's."""
    if split:
        monkeypatch.setenv("GMLX_KQ_SDPA_SPLIT", split)  # (past 64 splits: the other merge)
    from gmlx_amd import ops
    rows = [(1, 5000), (40, 3000), (2, 900)]
    b = Batch(rows, Hq, Hkv, D, 16, BF16, q8=q8, seed=D)
    q = torch.ones(b.T, Hq, D, dtype=BF16, device="cuda")
    k, v = b.pool
    for r in range(len(rows)):  # the first 640 keys score 1000 below the others
        for t in range(0, 640, 16):
            page = int(b.table[r, t // 16])
            if q8:
                k[page], b.scales["k_scales"][page], b.scales["k_biases"][page] = 0, 0.0, -1000 * D ** -0.5
            else:
                k[page] = -1000 * D ** -0.5
    clean = b.run(q=q)
    assert torch.isfinite(clean).all()
    for r in range(len(rows)):
        page = int(b.table[r, 1])
        if q8:
            b.scales["v_biases"][page, 0, 3, 0] = float("nan")
        else:
            v[page, 0, 3, 5] = float("nan")
    _say("far NaN", D, q8, split)
    out = b.run(q=q)
    G, dims = Hq // Hkv, slice(0, 64) if q8 else slice(5, 6)
    assert torch.isnan(out[:, :G, dims]).all()
    out[:, :G, dims] = clean[:, :G, dims]
    assert torch.equal(out, clean)


def test_write_8bit_ranges_past_fp32():
    """bf16 groups whose largest and smallest value are further apart than fp32's
    largest: finite, and quantised as any other."""
    from gmlx_amd import ops
    (k, v), sc = _pool((2, 1, 16, 128), BF16, True, "head")
    x = torch.rand(9, 1, 128, dtype=torch.float64, generator=torch.Generator().manual_seed(1)) * 6e38 - 3e38
    x[:, :, 64:] /= 4  # (a range that fp32 holds)
    x[:, :, 3], x[:, :, 7] = 3.2e38, -3.2e38
    x = x.to(BF16)
    slots = torch.arange(9, dtype=torch.int32, device="cuda")
    _say("wide range")
    ops.paged_write(x.cuda(), x.cuda(), k, v, slots, **sc)
    got = ops.paged_read(k, v, slots, **sc)
    _, want_s, want_b = _quantised(x, BF16)
    for pool, name, back in ((k, "k", got[0]), (v, "v", got[1])):
        q = pool[0, :, :9].transpose(0, 1).cpu().unflatten(-1, (-1, 64)).double()
        s, b = (sc[name + t][0, :, :9].transpose(0, 1).cpu() for t in ("_scales", "_biases"))
        assert torch.equal(b, want_b) and torch.isfinite(s.float()).all()
        s, ws, b = s.double()[..., None], want_s.double()[..., None], b.double()[..., None]
        assert ((s - ws).abs() <= ws * torch.finfo(BF16).eps).all()
        ideal = ((x.double().unflatten(-1, (-1, 64)) - b) / s).clamp(0, 255)
        assert ((q - ideal).abs() <= 0.5 + 255 * 2.0 ** -22).all()
        val = (q * s + b).flatten(-2)
        assert ((back.cpu().double() - val).abs() <= val.abs() * (HALF[BF16] + 2.0 ** -23)).all()


def test_writes_to_pools_that_repeat_places_are_refused():
    from gmlx_amd import KQError, ops
    x = torch.ones(3, 2, 128, dtype=F16, device="cuda")
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    base = torch.zeros(2, 4, 1, 16, 128, dtype=F16, device="cuda")
    one = torch.zeros(4, 2, 16, 128, dtype=F16, device="cuda")
    for k, v in ((base[0].expand(4, 2, 16, 128), base[1].expand(4, 2, 16, 128)), (one, one)):
        with pytest.raises(KQError):
            ops.paged_write(x, x, k, v, slots)
        assert not k.any()
        ops.paged_read(k, v, slots)
    # layouts that interleave without sharing are taken
    for layout in ("head", "token", "mixed"):
        (k, v), _ = _pool((4, 2, 16, 128), F16, False, layout)
        ops.paged_write(x, x, k, v, slots)
        assert int(k.sum()) == int(v.sum()) == 3 * 2 * 128
    (k, v), _ = _pool((1, 1, 16, 64), F16, False, "token")
    ops.paged_write(x[:, :1, :64], x[:, :1, :64], k, v, slots)
    assert int(k.sum()) == 3 * 64


@pytest.mark.parametrize("D,Hq,Hkv,q8", [(64, 4, 2, False), (128, 8, 2, False), (128, 8, 2, True), (256, 4, 2, False)])
def test_scale_of_zero_with_large_products(D, Hq, Hkv, q8):
    """0 weighs all keys alike, products near fp32's largest too."""
    b = Batch([(1, 300), (40, 333)], Hq, Hkv, D, 16, BF16, q8=q8, seed=D, spread=1e17)
    q = b.q.cuda() * 1e17
    b.scale = 0.0
    _say("zero scale", D, q8)
    assert torch.equal(b.run(q=q), b.run(q=torch.zeros_like(q)))


def test_plan_sizes_past_32_bits_are_refused():
    """And not cut to their low bits."""
    from gmlx_amd import ops
    i32 = dict(dtype=torch.int32, device="cuda")
    one, table = torch.ones(1, **i32), torch.zeros(1, 4, **i32)
    for page, tokens in ((2 ** 32 + 16, 4), (16, 2 ** 31), (16, 2 ** 32 + 4)):
        with pytest.raises(ValueError, match="paged_plan"):
            ops.paged_plan(one, one, table, one, one, page, tokens)


def test_plan_of_rows_that_share_pages():
    """Rows with a common prefix of whole pages: each ended by keeping the shared
    tokens and a length of 0 by hand, the last one by keeping 0; every page is on
    the stack once."""
    table = np.array([[4, 2, 0, -1, -1], [4, 2, 3, 1, -1], [4, 2, 5, -1, -1]], np.int32)
    stack, count, seq = np.full(6, -9, np.int32), 0, [40, 52, 33]
    for keep, ended in (([40, 32, 33], 1), ([40, 0, 32], 2), ([0, 0, 0], 0)):
        got = _check_plan(seq, [0, 0, 0], table, stack, count, 16, 3, keep)
        seq, count, table, stack = got[1].tolist(), int(got[4][0]), got[6], got[7]
        seq[ended] = 0
        held = {int(p) for b, s in enumerate(seq) for p in table[b, :-(-s // 16)]}
        assert sorted([*held, *stack[:count]]) == list(range(6))


@pytest.mark.parametrize("D,q8", [(64, False), (128, False), (128, True), (256, True), (512, False)])
def test_sixty_four_query_heads_a_kv_head(D, q8):
    """The most there are: rows of one token are chunks then, in 16 and 8 bits."""
    b = Batch([(1, 1), (1, 700), (5, 90), (0, 3), (1, 2100)], 64, 1, D, 32, BF16, q8=q8, seed=D)
    if q8:  # (chunks round a probability times the value, not the centred one)
        b.err = [np.maximum(e, np.abs(v)) for e, v in zip(b.err, b.v)]
    _say("64 heads", D, q8)
    b.check(b.run())
    b.check(b.run(max_q=5, max_kv=2100))
