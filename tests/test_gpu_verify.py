"""Drafted tokens verified on the GPU against fp64 numpy: whole numbers, so equal.
(Two fp64 computations disagree where a border of the running sum and the draw are
within some 10^-13 of each other: inputs are random, or sums exact.)"""
import numpy as np
import pytest
import torch

from oracle import step as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _say(*a):
    print(*a, flush=True)


def _case(ns, V, dt, pt, seed, spread=3.0, near=0.5, temp=1.0):
    """Logits of ragged rows, drafts drawn from a model near the target's."""
    rng = np.random.default_rng(seed)
    T, B = int(sum(ns)), len(ns)
    logits = torch.from_numpy(rng.normal(0, spread, (T, V))).to(dt)
    other = logits.double().numpy() + rng.normal(0, near, (T, V))
    other = other / (temp if temp > 0 else 1.0)
    p = np.exp(other - other.max(1, keepdims=True)) if T else other
    p = p / p.sum(1, keepdims=True)
    tokens = np.zeros(T, np.int64)
    for t in range(T - 1):
        tokens[t + 1] = np.searchsorted(np.cumsum(p[t]), rng.random() * 0.999999)
    return dict(logits=logits.cuda(), tokens=torch.tensor(np.minimum(tokens, V - 1), dtype=torch.int32, device="cuda"),
                cu=torch.tensor(np.concatenate([[0], np.cumsum(ns)]), dtype=torch.int32, device="cuda"),
                uniforms=torch.from_numpy(rng.random(T).astype(np.float32)).cuda(),
                draws=torch.from_numpy(rng.random(B).astype(np.float32)).cuda(),
                draft_probs=None if pt is None else torch.from_numpy(p).to(pt).cuda(), temperature=temp,
                kv_lens=torch.tensor([n + 3 for n in ns], dtype=torch.int32, device="cuda"))


def _want(c):
    at = lambda x: None if x is None else x.double().cpu().numpy() if x.is_floating_point() else x.cpu().numpy()  # noqa: E731
    temp = c["temperature"]
    return ref.verify(at(c["logits"]), at(c["tokens"]), at(c["cu"]), at(c["uniforms"]), at(c["draws"]),
                      at(c["draft_probs"]), temp if not isinstance(temp, torch.Tensor) else at(temp), at(c["kv_lens"]))


def _check(c):
    from gmlx_amd import ops
    got = ops.verify_drafts(**c)
    want = _want(c)
    assert got.accepted.tolist() == want[0]
    assert got.tokens.tolist() == want[1]
    assert (got.keep_lens is None and want[2] is None) or got.keep_lens.tolist() == want[2]
    return got


@pytest.mark.parametrize("dt,pt", [(F16, None), (BF16, F32), (F32, F32), (F16, F16), (BF16, BF16), (F32, BF16), (F16, F32)])
@pytest.mark.parametrize("V", [1, 2, 7, 33, 1000, 2047, 2049, 8193, 50001])
def test_verify(V, dt, pt):
    rng = np.random.default_rng(V)
    ns = [1, 5, 0, 3, 9, 2, 1, 4, 0] + rng.integers(0, 7, 5 if V > 9000 else 40).tolist()
    _say("verify", V, dt, pt)
    for temp in (1.0, 0.0, 0.6, 2.5):
        _check(_case(ns, V, dt, pt, V + int(10 * temp), temp=temp))


def test_a_large_batch_takes_long_slices():
    for V, B, dt, pt in ((32000, 300, BF16, None), (9001, 500, F32, F16)):
        rng = np.random.default_rng(B)
        _say("large", V, B)
        _check(_case(rng.integers(1, 4, B).tolist(), V, dt, pt, B))


@pytest.mark.parametrize("B", [512, 513])
def test_rows_at_the_border_of_a_launch(B):
    """9 slices, 3 workgroups a row: 1536 find their rows' ends themselves, 1539 do not."""
    ns = np.random.default_rng(B).integers(0, 4, B).tolist()
    _say("border", B)
    _check(_case(ns, 9001, F32, F32, B, near=2.0))


def _late_case(ns, V, dt, pt, seed, temp=1.0):
    """Rows whose likely tokens lie in the slices past the 64th (of 4 KB of logits), with about as many drafts that
    stand there as are refused there."""
    rng = np.random.default_rng(seed)
    T, B, late = int(sum(ns)), len(ns), 64 * 4096 // dt.itemsize
    assert V > late
    x = rng.normal(0, 1, (T, V)).astype(np.float32)
    likely = np.stack([late + rng.permutation(V - late)[:min(24, V - late)] for _ in range(T)])
    at = np.arange(T)[:, None]
    x[at, likely] = 10 + rng.normal(0, 1, likely.shape)
    x[np.arange(T), rng.integers(0, late, T)] = 11  # and one before
    logits = torch.from_numpy(x).to(dt)
    other = logits.double().numpy()
    other[at, likely] += rng.normal(0, 1.0, likely.shape)
    other = np.exp((other - other.max(1, keepdims=True)) / (temp if temp > 0 else 1.0))
    p = other / other.sum(1, keepdims=True)
    tokens = np.zeros(T, np.int64)
    for t in range(T - 1):
        tokens[t + 1] = logits[t].argmax() if temp == 0 and t % 2 else np.searchsorted(np.cumsum(p[t]), rng.random() * 0.999999)
    return dict(logits=logits.cuda(), tokens=torch.tensor(tokens, dtype=torch.int32, device="cuda"),
                cu=torch.tensor(np.concatenate([[0], np.cumsum(ns)]), dtype=torch.int32, device="cuda"),
                uniforms=torch.from_numpy(rng.random(T).astype(np.float32)).cuda(),
                draws=torch.from_numpy(rng.random(B).astype(np.float32)).cuda(),
                draft_probs=None if pt is None else torch.from_numpy(p).to(pt).cuda(), temperature=temp,
                kv_lens=torch.tensor([n + 3 for n in ns], dtype=torch.int32, device="cuda"))


# slices: 65 and 69 of 1024 values, 65 and 75 of 2048 (one value in the last of the first of each)
@pytest.mark.parametrize("V,dt", [(65537, F32), (70001, F32), (131073, F16), (152064, BF16)])
@pytest.mark.parametrize("pt", [None, F32, F16])
@pytest.mark.parametrize("temp", [1.0, 0.7, 0.0])
def test_drafts_past_the_64th_slice(V, dt, pt, temp):
    _say("late", V, dt, pt, temp)
    ns = [2, 3, 1, 5, 4, 2, 2, 3, 6, 2, 2, 1, 3, 2]
    c = _late_case(ns, V, dt, pt, V + int(10 * temp), temp)
    got = _check(c)
    late = 64 * 4096 // dt.itemsize
    cu, tokens, acc = (x.tolist() for x in (c["cu"], c["tokens"], got.accepted))
    fell = sum(tokens[cu[b] + 1 + acc[b]] >= late for b in range(len(ns)) if acc[b] < ns[b] - 1)
    stood = lambda acc: sum(tokens[cu[b] + 1 + i] >= late for b in range(len(ns)) for i in range(acc[b]))  # noqa: E731
    if V in (65537, 131073):  # (whose last slice is one token)
        return
    assert fell >= 2 and sum(t >= late for t in got.tokens.tolist()) >= 5
    if pt is None and temp:  # (of 24 likely tokens a lone draft stands once in some 24 times: with smaller numbers too)
        c["uniforms"] *= 0.05
        got = _check(c)
    assert stood(got.accepted.tolist()) >= 3


@pytest.mark.parametrize("B", [90, 91])
def test_many_rows_of_drafts_past_the_64th_slice(B):
    """17 workgroups a row: 1530 find their rows' ends themselves, 1547 do not."""
    _say("late", B)
    ns = np.random.default_rng(B).integers(1, 4, B).tolist()
    _check(_late_case(ns, 66000, F32, F32, B, 0.7))


@pytest.mark.parametrize("pt", [None, BF16])
def test_a_vocabulary_of_thousands_of_slices(pt):
    V = (1 << 24) + 5  # 8193 slices, five tokens in the last
    rng = np.random.default_rng(3)
    x = torch.randn(3, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    x[:, V - 3] = 16.0
    x[0, [5, 1 << 23]] = 15.0
    x = x.to(BF16)
    p = None
    if pt is not None:
        p = torch.softmax(x.float(), 1).to(pt)
        p[:, V - 3] *= 1.5
    for temp in (1.0, 0.0):
        for draft, draw in ((V - 3, 0.0), (V - 3, 0.999), (7, 0.3), (V, 0.97), (1 << 23, 0.5)):
            c = dict(logits=x, tokens=torch.tensor([0, V - 3, draft], dtype=torch.int32, device="cuda"),
                     cu=torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                     uniforms=torch.tensor([0.0, rng.random(), 0.0], device="cuda").float(),
                     draws=torch.tensor([draw], device="cuda"), draft_probs=p, temperature=temp,
                     kv_lens=torch.tensor([9], dtype=torch.int32, device="cuda"))
            _say("vocabulary", pt, temp, draft, draw)
            _check(c)


def test_equal_logits_in_slices_of_one_lane():
    """The largest logit in slices 3, 67 and 131 (one lane's), 130 (an earlier lane's) and within a slice twice."""
    from gmlx_amd import ops
    V = 140 * 1024
    spots = [[3, 67, 131], [67, 131], [130, 131], [66, 67], [131], [64, 2 + 64], [139]]
    x = torch.randn(len(spots), V, device="cuda")
    for t, where in enumerate(spots):
        for s in where:
            x[t, [s * 1024 + 77, s * 1024 + 900]] = 9.0
    want = [w[0] * 1024 + 77 for w in spots]
    n = len(spots)
    r = ops.verify_drafts(x, torch.tensor([0] + want[:-1], dtype=torch.int32, device="cuda"),
                          torch.tensor([0, n], dtype=torch.int32, device="cuda"), temperature=0)
    assert r.accepted.tolist() == [n - 1] and r.tokens.tolist() == [want[-1]]


def test_a_lone_draft_holds_its_late_slice():
    """A refused draft with all but a millionth of the weight of a slice past the 64th, or all of the row's."""
    from gmlx_amd import ops
    V, d = 70001, 66 * 1024 + 5
    for others in (-20.0, -60.0, -float("inf")):
        x = torch.full((2, V), others, device="cuda")
        x[0, d], x[0, 3] = 4.0, -12.0
        x[0, d + 1] = -18.0
        kw = dict(tokens=torch.tensor([0, d], dtype=torch.int32, device="cuda"), uniforms=torch.ones(2, device="cuda"))
        for draw in (0.0, 0.3, 0.9, 0.99999, 0.9999999):
            c = dict(logits=x, cu=torch.tensor([0, 2], dtype=torch.int32, device="cuda"),
                     draws=torch.tensor([draw], device="cuda"), draft_probs=None, temperature=1.0,
                     kv_lens=torch.tensor([9], dtype=torch.int32, device="cuda"), **kw)
            got = _check(c)
            assert got.accepted.tolist() == [0] and got.tokens.tolist() != [d]


@pytest.mark.parametrize("V,share", [(1500, 2e-6), (1500, 1e-4), (1500, 0.05), (9000, 3e-6), (150000, 2e-4)])
def test_draws_behind_a_refused_draft_of_nearly_all_the_weight(V, share):
    """The rest of a row whose lone draft holds all but `share` of the weight is summed by itself: taken off the whole,
    it would keep the whole's error, 10^-16 and more of it.  Draws are the numbers nearest to a border of the rest, of
    which they are 10^-8 apart at most."""
    from gmlx_amd import ops
    n = 300
    rng = np.random.default_rng(V)
    x = rng.normal(0, 1, V)
    x = torch.from_numpy(x - np.log(np.exp(x).sum() / share)).float()  # (a sum of `share` beside the draft's 1)
    d = V // 3
    x[d] = 0.0
    w = np.exp(x.numpy().astype(np.longdouble))
    w[d] = 0
    run = np.cumsum(w)
    border = run / run[-1]
    draw = border.astype(np.float32)
    gap = np.abs(draw - border)
    ok = np.nonzero((gap > _APART) & (draw < 1) & (w > 0))[0]
    ok = ok[np.argsort(gap[ok])[:n]]  # the nearest
    n = len(ok)
    draws = draw[ok]
    want = np.searchsorted(run, draws.astype(np.longdouble) * run[-1], side="right")
    tokens = torch.tensor([0, d] * n, dtype=torch.int32, device="cuda")
    r = ops.verify_drafts(x.cuda()[None].expand(2 * n, V), tokens, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"),
                          torch.ones(2 * n, device="cuda"), torch.from_numpy(draws).cuda())
    assert r.accepted.tolist() == [0] * n
    got = r.tokens.cpu().numpy()
    _say("rest", V, share, float(gap[ok].min()), float(gap[ok].max()), int((got != want).sum()), "of", n)
    assert np.array_equal(got, want)


def test_drafts_of_all_kinds_of_agreement():
    """Models that agree (all stand) and that do not (the first falls), long drafts."""
    for near, spread in ((0.0, 4.0), (8.0, 4.0), (0.1, 0.0)):
        _say("near", near)
        got = _check(_case([70, 1, 130, 6], 300, F32, F32, 5, spread=spread, near=near))
        if near == 0.0:
            assert got.accepted.tolist() == [69, 0, 129, 5]


# A border and a draw that is further than this from it (of the whole): weights good to 4e-14, two of them in a quotient,
# and some 200 roundings of 2^-53 in a running sum of the kernel's come to 1.1e-13; the references below are in 80 bits.
_APART = np.longdouble(1e-12)


@pytest.mark.parametrize("temp", [0.7, 0.8])
def test_draws_at_a_temperature_that_32_bits_do_not_hold(temp):
    """60000 draws from one flat row: with the temperature rounded to 32 bits, off by 1.7e-8 and 1.5e-8 of itself, weights
    are off by that times their distance from the largest, and some ten draws fall on another side of some border."""
    from gmlx_amd import ops
    B, V = 60000, 152064
    rng = np.random.default_rng(int(10 * temp))
    x = torch.from_numpy(rng.normal(0, 3, V)).half()
    draws = rng.random(B).astype(np.float32)
    w = x.numpy().astype(np.longdouble)
    w = np.exp((w - w.max()) / np.longdouble(temp))
    run = np.cumsum(w)
    at = draws.astype(np.longdouble) * run[-1]
    want = np.searchsorted(run, at, side="right")
    near = np.minimum(np.abs(run[want] - at), np.abs(run[np.maximum(want - 1, 0)] - at)) < _APART * run[-1]
    assert near.sum() < 10
    _say("draws", temp, int(near.sum()), "left out")
    r = ops.verify_drafts(x.cuda()[None].expand(B, V), torch.zeros(B, dtype=torch.int32, device="cuda"),
                          torch.arange(B + 1, dtype=torch.int32, device="cuda"), torch.zeros(B, device="cuda"),
                          torch.from_numpy(draws).cuda(), temperature=temp)
    got = r.tokens.cpu().numpy()
    assert np.array_equal(got[~near], want[~near]), int((got != want).sum())


@pytest.mark.parametrize("temp", [0.6, 0.7, 0.8, 1.0])
def test_drafts_whose_uniform_is_the_nearest_number_to_their_border(temp):
    """u is p_d rounded to 32 bits, above or below it by up to 6e-8 of it; weights off by 2e-8 times a distance of some
    ten logits would judge many of them the other way."""
    from gmlx_amd import ops
    n, V = 400, 1000
    rng = np.random.default_rng(7)
    x = torch.from_numpy(rng.normal(0, 3, (n, V))).half()
    d = rng.integers(0, V, n)
    w = x.numpy().astype(np.longdouble)
    w = np.exp((w - w.max(1, keepdims=True)) / np.longdouble(temp))
    p = w[np.arange(n), d] / w.sum(1)
    u = p.astype(np.float32)
    kept = (np.abs(u - p) > _APART * p) & (u > 1e-30)
    assert kept.sum() > 0.9 * n
    tokens, uniforms = np.zeros((n, 2), np.int32), np.zeros((n, 2), np.float32)
    tokens[:, 1], uniforms[:, 0] = d, u
    r = ops.verify_drafts(x.cuda().repeat_interleave(2, 0), torch.from_numpy(tokens.reshape(-1)).cuda(),
                          torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"),
                          torch.from_numpy(uniforms.reshape(-1)).cuda(), torch.full((n,), 0.5, device="cuda"), temperature=temp)
    got = r.accepted.cpu().numpy()
    assert np.array_equal(got[kept], (u < p).astype(np.int32)[kept]), int((got != (u < p)).sum())


@pytest.mark.parametrize("temp", [1e-310, 1e-60, 1e-40, 1e39, 1e60, 1e308])
def test_temperatures_past_the_ends_of_32_bits(temp):
    for dt, pt, near in ((F16, None, 0.5), (F32, F32, 0.01)):
        c = _case([4, 3, 1, 5, 2, 6], 5000, dt, pt, 12, near=near)
        c["temperature"] = temp
        _check(c)


def test_temperatures_by_row():
    c = _case([4, 3, 1, 5, 2, 6], 5000, BF16, F32, 11)
    c["temperature"] = torch.tensor([1.0, 0.0, -1.0, 0.3, float("nan"), 1e-30], device="cuda")
    _check(c)


def test_equal_logits_go_to_the_lowest_and_exact_sums():
    """Equal weights sum exactly: the draw of k / V starts token k."""
    from gmlx_amd import ops
    V = 4096
    B = 64
    x = torch.zeros(B, V, device="cuda")
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    k = torch.arange(B, device="cuda") * 63
    r = ops.verify_drafts(x, torch.zeros(B, dtype=torch.int32, device="cuda"), cu, torch.zeros(B, device="cuda"),
                          (k.double() / V).float())
    assert r.tokens.tolist() == k.tolist() and r.accepted.tolist() == [0] * B and r.keep_lens is None
    x[:, 7] = x[:, 4000] = 2.0
    r = ops.verify_drafts(x.bfloat16(), torch.zeros(B, dtype=torch.int32, device="cuda"), cu, temperature=0)
    assert r.tokens.tolist() == [7] * B


@pytest.mark.parametrize("pt", [None, F32])
def test_draws_at_the_ends(pt):
    c = _case([3, 1, 4, 2, 5], 2500, F16, pt, 21)
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0):
        for r in (0.0, 1.0 - 2.0 ** -24, 1.0, 1.5, -1.0):
            c["uniforms"].fill_(u)
            c["draws"].fill_(r)
            _say("ends", u, r)
            if pt is None and r < 1:
                _check(c)
            elif r < 1 - 2.0 ** -23:
                _check(c)
            else:  # (a border within 10^-13 of the whole is any of the last tokens': one with weight)
                from gmlx_amd import ops
                got = ops.verify_drafts(**c)
                assert got.accepted.tolist() == _want(c)[0] and all(0 <= t < 2500 for t in got.tokens.tolist())


def test_a_refused_draft_without_weight_takes_none_along():
    """A draft, and all its slice, below any weight: a draw of 1 ends before them."""
    from gmlx_amd import ops
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.zeros(2, 5000, device="cuda").bfloat16()
    x[:, 4096:] = -10000.0
    f = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    for draw, want in ((1.0, 4095), (0.5, 2048), (2.0, 4095)):
        r = ops.verify_drafts(x, i32(0, 4500), i32(0, 2), f(0.0, 0.0), f(draw))
        assert (r.accepted.tolist(), r.tokens.tolist()) == ([0], [want])


def test_logits_and_probabilities_that_are_not_finite():
    nan, inf = float("nan"), float("inf")
    for temp in (1.0, 0.0, 0.5):
        for dt in (F32, F16, BF16):
            c = _case([3, 3, 2, 4, 1, 2, 3], 3000, dt, F32, 31, temp=temp)
            x, p = c["logits"], c["draft_probs"]
            x[0, ::2] = -inf
            x[1, 5] = nan
            x[3] = -inf                     # nothing to take
            x[6, :] = nan
            x[8, 77] = inf
            x[9, [3, 2999]] = inf
            x[12] = -inf
            x[12, 1234] = -5.0              # one token only
            x[13, :2999] = -inf
            p[1, 4:900] = nan
            p[4] = -1.0
            p[9] = 0.0
            p[10, 7] = inf
            c["tokens"][2], c["tokens"][10] = 3000, -5  # no tokens
            _say("odd", temp, dt)
            _check(c)
            c["draft_probs"] = None
            _check(c)


def test_probabilities_equal_to_the_targets_leave_no_rest():
    """Nothing is left beside q: the target's own."""
    from gmlx_amd import ops
    V = 1024
    x = torch.zeros(2, V, device="cuda")
    p = torch.full((2, V), 1.0 / V, device="cuda")  # exact
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    r = ops.verify_drafts(x, i32(0, 9), i32(0, 2), torch.ones(2, device="cuda"), torch.tensor([0.5], device="cuda"), p)
    assert (r.accepted.tolist(), r.tokens.tolist()) == ([0], [512])


def test_kept_tokens_follow_the_target():
    """The first token after a step (a draft that stands, or the token in its
    place) has the target's distribution: 40000 rows, five deviations."""
    from gmlx_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(7)
    B, V = 40000, 6
    p = torch.tensor([0.4, 0.05, 0.25, 0.0, 0.2, 0.1], device="cuda")
    q = torch.tensor([0.1, 0.5, 0.15, 0.05, 0.0, 0.2], device="cuda")
    x = p.log().repeat(2 * B, 1)
    drafts = torch.multinomial(q, B, replacement=True, generator=gen).int()
    tokens = torch.stack([torch.zeros_like(drafts), drafts], 1).reshape(-1).contiguous()
    cu = torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device="cuda")
    u, r = torch.rand(2 * B, device="cuda", generator=gen), torch.rand(B, device="cuda", generator=gen)
    for probs in (q.expand(2 * B, V), None):
        d = tokens if probs is not None else torch.where(torch.arange(2 * B, device="cuda") % 2 == 1, 2, 0).int()
        got = ops.verify_drafts(x, d, cu, u, r, draft_probs=probs)
        first = torch.where(got.accepted == 1, d[1::2], got.tokens).long()
        share = torch.bincount(first, minlength=V).double() / B
        room = 5 * (p.double() * (1 - p.double()) / B).sqrt() + 1e-9
        assert ((share - p.double()).abs() <= room).all(), share


def test_padding_strides_and_the_same_bits_again():
    """Rows behind the last sequence are not read; rows of a wider matrix, rows at
    odd addresses, one row for all."""
    from gmlx_amd import ops
    c = _case([2, 4, 1, 3], 1003, BF16, F32, 41)
    want = _check(c)
    wide = torch.full((14, 1009), float("nan"), dtype=BF16, device="cuda")
    wide[:10, 3:1006] = c["logits"]
    probs = torch.full((14, 1007), float("nan"), device="cuda")
    probs[:10, 1:1004] = c["draft_probs"]
    pad = lambda x, v: torch.cat([x, torch.full((4,), v, dtype=x.dtype, device="cuda")])  # noqa: E731
    got = ops.verify_drafts(wide[:, 3:1006], pad(c["tokens"], -1), c["cu"], pad(c["uniforms"], float("nan")), c["draws"],
                            probs[:, 1:1004], kv_lens=c["kv_lens"])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    one = c["logits"][:1].expand(10, 1003)
    c["logits"] = one
    _check(c)
    c["logits"] = c["logits"].t().contiguous().t()  # columns together: copied
    _check(c)


def test_logits_past_32_bits_of_bytes():
    """Rows whose byte offsets pass 2^32, many of them."""
    from gmlx_amd import ops
    T, V = 15000, 152064
    x = torch.zeros(T, V, dtype=F16, device="cuda")
    at = (torch.arange(T, device="cuda") * 7919) % V
    x[torch.arange(T, device="cuda"), at] = 30.0
    cu = torch.arange(T + 1, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(T, dtype=torch.int32, device="cuda")
    _say("past 32 bits")
    r = ops.verify_drafts(x, tokens, cu, temperature=0)
    assert torch.equal(r.tokens.long(), at)
    # (30 above the rest of V: 1 - V e^-30 of the weight)
    r = ops.verify_drafts(x, tokens, cu, torch.zeros(T, device="cuda"), torch.full((T,), 0.5, device="cuda"))
    assert torch.equal(r.tokens.long(), at)


def test_no_rows():
    from gmlx_amd import ops
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda n: torch.zeros(n, device="cuda")  # noqa: E731
    r = ops.verify_drafts(torch.zeros(0, 50, device="cuda"), z(0), z(4), f(0), f(3), kv_lens=z(3) + 5)
    assert (r.accepted.tolist(), r.tokens.tolist(), r.keep_lens.tolist()) == ([0] * 3, [-1] * 3, [5] * 3)
    r = ops.verify_drafts(torch.zeros(4, 50, device="cuda"), z(4), z(1), f(4), f(0))
    assert r.accepted.numel() == 0 and r.tokens.numel() == 0


def test_captured_and_replayed():
    """Two graphs captured on one stream, replayed in turn beside eager calls."""
    from gmlx_amd import ops
    cs = [_case([3, 5, 1], 9000, BF16, F32, 51), _case([2] * 9, 3001, F32, None, 52, temp=0.7)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for c in cs:
            ops.verify_drafts(**c)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(ops.verify_drafts(**c))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(4):
        for c, g, o in zip(cs, graphs, outs):
            c["draws"].copy_(torch.rand_like(c["draws"]))
            c["uniforms"].copy_(torch.rand_like(c["uniforms"]))
            g.replay()
            torch.cuda.synchronize()
            want = _check(c)
            for a, b in zip(o, want):
                assert torch.equal(a, b)


def test_refusals():
    from gmlx_amd import ops
    base = _case([2, 3], 100, F16, F32, 61)
    for bad in (dict(logits=base["logits"][0]), dict(logits=base["logits"].cpu()), dict(logits=base["logits"].double()),
                dict(tokens=base["tokens"][:3]), dict(tokens=base["tokens"].long()), dict(cu=base["cu"].long()),
                dict(uniforms=None), dict(draws=None), dict(uniforms=base["uniforms"].double()), dict(draws=base["draws"][:1]),
                dict(draft_probs=base["draft_probs"][:, :99]), dict(draft_probs=base["draft_probs"].double()),
                dict(temperature=-0.5), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(temperature=torch.ones(3, device="cuda")), dict(kv_lens=base["kv_lens"][:1])):
        with pytest.raises(ValueError):
            ops.verify_drafts(**{**base, **bad})
