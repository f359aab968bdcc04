"""Attention of new tokens through a window and a row's first keys, over a paged
cache whose pages in between are gone, against fp64 numpy."""
import numpy as np
import pytest
import torch

from oracle import step as ref
from test_gpu_paged import HALF, Batch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _say(*a):
    print(*a, flush=True)


class Windowed(Batch):
    """Rows whose pages between the sinks and the first new token's window are no
    entries of the table, and whose places there hold NaN."""

    def __init__(self, rows, Hq, Hkv, D, P, dt, window, sinks, **kw):
        super().__init__(rows, Hq, Hkv, D, P, dt, **kw)
        self.window, self.sinks, self.P = window, sinks, P
        tab = self.table.cpu().numpy()
        for b, (n, kv) in enumerate(rows):
            first = max(kv - n + 1 - window, 0) // P
            kept = -(-sinks // P)
            for p in range(kept, min(first, tab.shape[1])):
                tab[b, p] = -1 if p % 2 else 2 ** 31 - 1
        self.table = torch.from_numpy(tab).cuda()

    def run(self, **kw):
        from gmlx_amd import ops
        kw = {"window": self.window, "sinks": self.sinks, **kw}
        q = kw.pop("q") if "q" in kw else self.q.cuda()
        return ops.sdpa_paged(q, *self.pool, self.table, self.kv_lens, self.cu_q, self.scale, **self.scales, **kw)

    def check(self, out, max_q=None, max_kv=None):
        """As the attention without a window is checked, over the keys seen: within
        the output's rounding, the probabilities' and the 32-bit work.  A rounded
        probability (1 + d) p, |d| <= u, multiplies the centred integers of an 8-bit
        row of few columns, d p s (q - 128), and in chunks the value itself, d p (s q +
        b), as two halves of u^2 |v| rest: so u times the mean of the larger of
        |s (q - 128)| and |v|, and u^2 of it again."""
        u = HALF[self.dt]
        got = out.double().cpu().numpy()
        for b, (n, kv) in enumerate(self.rows):
            m = n if max_q is None else min(n, max_q)
            if not m:
                continue
            q = self.q[self.cu[b]:self.cu[b] + m].double().numpy()
            keys = slice(0, kv if max_kv is None else min(kv, max_kv))
            k, v, err = self.k[b][:, keys], self.v[b][:, keys], np.maximum(self.err[b], np.abs(self.v[b]))[:, keys]
            want, far = ref.window_attention(q, k, v, n, self.scale, self.window, self.sinks, err, kv)
            _, mean = ref.window_attention(q, k, v, n, self.scale, self.window, self.sinks, None, kv)
            seen = min(kv, self.window + self.sinks)
            smax = 1.5 * self.scale * np.abs(q).sum(-1).max() * max(1.0, np.abs(k).max() if k.size else 1.0)
            f32 = 2.0 ** -24 * (2 * (q.shape[-1] + 8) * smax + 2 * seen + 16)
            room = u * np.abs(want) + u * (1 + 2 * u) * far + f32 * (mean + far) + 1e-7
            d = np.abs(got[self.cu[b]:self.cu[b] + m] - want)
            assert np.isfinite(d).all() and (d <= room).all(), (b, n, kv, (d / room).max())


ROWS = [(1, 1), (1, 15), (0, 40), (1, 16), (1, 33), (3, 3), (7, 7 + 64), (0, 0), (5, 2), (2, 0), (1, 700), (40, 333),
        (1, 0), (2, 1500), (150, 700)]
SHAPES = [(128, 32, 8), (64, 8, 8), (96, 12, 3), (256, 16, 2), (128, 5, 1), (512, 8, 1), (64, 64, 2), (128, 48, 1)]
WINDOWS = [(1, 0), (1, 3), (5, 0), (16, 16), (17, 4), (64, 1), (100, 70), (256, 20), (333, 0), (4000, 4)]


@pytest.mark.parametrize("D,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("i", range(len(WINDOWS)))
def test_windows(D, Hq, Hkv, i):
    window, sinks = WINDOWS[i]
    dt = BF16 if i % 2 else F16
    _say("window", D, Hq, Hkv, window, sinks, dt)
    b = Windowed(ROWS, Hq, Hkv, D, 16, dt, window, sinks, seed=D + Hq + i)
    b.check(b.run())


@pytest.mark.parametrize("D,Hq,Hkv", [s for s in SHAPES if s[0] != 96])
@pytest.mark.parametrize("i", range(len(WINDOWS)))
def test_windows_8bit(D, Hq, Hkv, i):
    window, sinks = WINDOWS[i]
    dt = F16 if i % 2 else BF16
    _say("window8", D, Hq, Hkv, window, sinks, dt)
    b = Windowed(ROWS, Hq, Hkv, D, 32, dt, window, sinks, q8=True, seed=D + Hq + i)
    b.check(b.run())


@pytest.mark.parametrize("P,layout,q8", [(16, "head", False), (64, "token", False), (256, "mixed", False),
                                         (1024, "head", True), (128, "mixed", True)])
def test_long_rows(P, layout, q8):
    """Windows of many splits, behind many pages given back."""
    rows = [(1, 9000), (6, 6345), (1, 5000), (130, 7001), (1, 4099)]
    for window, sinks in ((4096, 4), (1000, 2000), (3001, 130)):
        _say("long", P, layout, q8, window, sinks)
        b = Windowed(rows, 8, 2, 128, P, BF16, window, sinks, q8=q8, layout=layout, seed=P)
        b.check(b.run())


@pytest.mark.parametrize("window,sinks", [(16382, 1), (16384, 0), (16385, 0), (16300, 200), (20000, 4)])
@pytest.mark.parametrize("Hq,Hkv,D,q8", [(8, 2, 128, False), (8, 2, 64, True), (4, 1, 256, False)])
def test_wide_windows(window, sinks, Hq, Hkv, D, q8):
    """On both sides of the line behind which splits go by the row: rows shorter than the window, at its end and past it."""
    rows = [(1, 1700), (1, window + 3), (3, 25000), (1, 600), (1, window - 1), (20, 16400), (1, 4097)]
    b = Windowed(rows, Hq, Hkv, D, 64, F16, window, sinks, q8=q8, seed=window)
    _say("wide", window, sinks, Hq, D, q8)
    out = b.run()
    b.check(out)
    from gmlx_amd import ops
    for i in (0, 2, 4):  # a row alone has its bits
        lo, hi = int(b.cu[i]), int(b.cu[i + 1])
        one = ops.sdpa_paged(b.q[lo:hi].cuda(), *b.pool, b.table[i:i + 1], b.kv_lens[i:i + 1],
                             torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"), b.scale, max_q=hi - lo,
                             max_kv=rows[i][1], window=window, sinks=sinks, **b.scales)
        assert torch.equal(one, out[lo:hi]), rows[i]


def test_a_window_past_every_row_is_none():
    for q8 in (False, True):
        rows = [(1, 700), (40, 333), (5, 2), (1, 5000), (130, 2100)]
        b = Windowed(rows, 8, 2, 128, 16, F16, 1 << 30, 3, q8=q8, seed=3)
        _say("past", q8)
        for window, sinks in ((1 << 30, 3), (5000, 0), (64, 1 << 30)):
            b.check(b.run(window=window, sinks=sinks))


@pytest.mark.parametrize("D,Hq,Hkv,q8", [(128, 32, 8, False), (128, 32, 8, True), (256, 16, 2, False), (64, 8, 8, False),
                                         (512, 8, 2, False)])
def test_row_equals_the_call_on_the_row_alone(D, Hq, Hkv, q8):
    from gmlx_amd import ops
    rows = [(1, 5000), (1, 130), (200, 1700), (4, 2600), (1, 1), (37, 37)]
    b = Windowed(rows, Hq, Hkv, D, 16, BF16, 700, 5, q8=q8, seed=9)
    full = b.run()
    assert torch.equal(full, b.run())
    for i, (n, kv) in enumerate(rows):
        lo, hi = int(b.cu[i]), int(b.cu[i + 1])
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        _say("alone", D, q8, n, kv)
        one = ops.sdpa_paged(b.q[lo:hi].cuda(), *b.pool, b.table[i:i + 1], b.kv_lens[i:i + 1], cu, b.scale, max_q=n,
                             max_kv=kv, window=700, sinks=5, **b.scales)
        assert torch.equal(one, full[lo:hi]), (n, kv)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("rows", [[(1, 500)], [(4, 300), (1, 90)], [(150, 900)], [(70, 2000), (1, 3000)]])
def test_cuts(rows, q8):
    """Of longer rows the first max_q tokens, and the first max_kv keys (also where
    they end before the window, or inside the sinks)."""
    for window, sinks in ((60, 4), (200, 30), (31, 0)):
        b = Windowed(rows, 8, 2, 128, 16, F16, window, sinks, q8=q8, seed=len(rows))
        most = max(kv for _, kv in rows)
        for max_kv in (most + 100, most - 10, most - window // 2, most // 2, 20, 3):
            _say("cut kv", rows, window, sinks, max_kv)
            b.check(b.run(max_kv=max_kv), max_kv=max_kv)
        n = max(n for n, _ in rows)
        for max_q in {max(1, n // 2), max(1, n - 1)}:
            out = torch.full_like(b.q.cuda(), 7.0)
            _say("cut q", rows, window, sinks, max_q)
            b.check(b.run(max_q=max_q, out=out), max_q=max_q)
            for i, (m, _) in enumerate(rows):
                assert (out[int(b.cu[i]) + min(m, max_q):int(b.cu[i + 1])] == 7).all()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,kv,Hq,D,window,sinks", [(1, 200, 8, 128, 50, 5), (5, 170, 8, 128, 21, 3), (40, 190, 8, 64, 30, 0),
                                                    (150, 400, 8, 128, 77, 20), (150, 400, 32, 128, 300, 4),
                                                    (60, 300, 4, 256, 64, 16), (30, 300, 4, 512, 40, 2)])
def test_values_outside_the_window(n, kv, Hq, D, window, sinks, dt):
    """Infinities and NaN in keys and values that a token does not see leave it as
    it is, whichever tokens beside it see them."""
    base = Windowed([(n, kv), (1, 20)], Hq, 2, D, 16, dt, window, sinks, seed=n)
    clean = base.run()
    k, v = base.pool
    P, before = 16, kv - n
    low = max(before + 1 - window, 0)
    for hit in sorted({low - 1, low, low + n // 2, before + n // 2, sinks - 1, sinks, kv - 1}):
        if hit < 0 or int(base.table[0, hit // P]) in (-1, 2 ** 31 - 1):
            continue
        page, off = int(base.table[0, hit // P]), hit % P
        for bad, what in ((float("inf"), "v"), (float("nan"), "v"), (float("nan"), "k")):
            _say("outside", hit, bad, what, n, kv, window, sinks, dt)
            pool = v if what == "v" else k
            was = pool[page, :, off].clone()
            pool[page, 1, off, 3] = bad
            out = base.run()
            pool[page, :, off] = was
            me = before + torch.arange(n)
            sees = (hit <= me) & ((hit > me - window) | (hit < sinks))
            half = Hq // 2
            assert torch.equal(out[n:], clean[n:]) and torch.equal(out[:n, :half], clean[:n, :half])
            assert torch.equal(out[:n][~sees], clean[:n][~sees])
            got = out[:n, half:][sees]
            if what == "k":
                assert torch.isnan(got).all()
            elif got.numel():
                col = got[..., 3].float()
                assert (torch.isnan(col) | (col == bad)).all()
                rest = [d for d in range(D) if d != 3]
                assert torch.equal(got[..., rest], clean[:n, half:][sees][..., rest])


@pytest.mark.parametrize("D,q8", [(128, False), (128, True), (256, False), (512, False)])
def test_pages_missing_in_the_window_and_among_the_sinks(D, q8):
    """Their keys are not seen; where none is left, zeros."""
    P, window, sinks = 16, 100, 40
    b = Windowed([(1, 700), (3, 90), (60, 500), (1, 17)], 8, 2, D, P, F16, window, sinks, q8=q8, seed=D)
    holes = {0: (0, 40), 1: (1, 3), 2: (2, 27, 30), 3: (0, 1)}
    tab = b.table.cpu().numpy()
    for row, pages in holes.items():
        for p in pages:
            tab[row, p] = -1 if p % 2 else 10 ** 6
    b.table = torch.from_numpy(tab).cuda()
    _say("holes", D, q8)
    out = b.run().double().cpu().numpy()
    for row, (n, kv) in enumerate(b.rows):
        keep = np.array([t // P not in holes[row] for t in range(kv)])
        for i in range(n):
            me = kv - n + i
            t = np.arange(kv)
            see = keep & (t <= me) & ((t > me - window) | (t < sinks))
            q = b.q[b.cu[row] + i:b.cu[row] + i + 1].double().numpy()
            got = out[b.cu[row] + i]
            if not see.any():
                assert (got == 0).all()
                continue
            k, v = b.k[row][:, see], b.v[row][:, see]
            err = np.maximum(b.err[row], np.abs(b.v[row]))[:, see]
            want, far = ref.window_attention(q, k, v, 1, b.scale, 10 ** 6, 0, err)
            # the output's and the probabilities' roundings, and 2^-16 for the 32-bit work of 140 keys
            assert (np.abs(got - want[0]) <= HALF[F16] * (np.abs(want[0]) + 1.01 * far[0]) + 2.0 ** -16 * far[0] + 1e-7).all()


@pytest.mark.parametrize("D,q8", [(128, False), (128, True), (256, False), (512, False)])
def test_output_in_place_and_rows_behind_the_last(D, q8):
    """The output may be the queries; rows behind the last sequence stay as they were."""
    b = Windowed([(1, 700), (0, 30), (70, 500), (2, 64), (0, 0)], 8, 2, D, 16, BF16, 90, 4, q8=q8, seed=D, pad=3)
    q = b.q.cuda()
    q[b.T:] = float("nan")
    want = b.run(q=q.clone(), out=torch.full_like(q, 7.0))
    assert (want[b.T:] == 7).all()
    b.check(want)
    got = b.run(q=q, out=q)
    assert got is q and torch.equal(q[:b.T], want[:b.T]) and torch.isnan(q[b.T:]).all()
    # strided queries and output
    wide = torch.full((b.T + 3, 8 * D + 64), 5.0, device="cuda").to(BF16)
    src = torch.zeros(b.T + 3, 8 * D + 8, device="cuda").to(BF16)
    src[:, :8 * D] = b.q.cuda().view(b.T + 3, -1)
    out = wide[:, 64:].view(b.T + 3, 8, D)
    b.run(q=src[:, :8 * D].view(b.T + 3, 8, D), out=out)
    assert torch.equal(out[:b.T], want[:b.T]) and (wide[:, :64] == 5).all() and (out[b.T:] == 5).all()


def test_captured_steps_through_a_window():
    b = Windowed([(1, 900), (5, 400), (60, 300)], 8, 2, 128, 16, BF16, 100, 4, seed=4)
    q = b.q.cuda()
    want = b.run(q=q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.run(q=q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = b.run(q=q)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(4):
        q.mul_(-0.75)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, b.run(q=q))
    assert not torch.equal(got, want)


def test_refusals():
    b = Windowed([(1, 40)], 8, 2, 128, 16, F16, 8, 0)
    for bad in (dict(window=0), dict(window=-1), dict(window=(1 << 30) + 1), dict(sinks=-1), dict(sinks=(1 << 30) + 1),
                dict(window=None, sinks=4)):
        with pytest.raises(ValueError):
            b.run(**bad)
