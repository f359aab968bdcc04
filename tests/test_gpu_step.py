"""A server's step over the paged cache, its operators together: pages and slots of
the step, queries and keys normed, rotated and stored, attention through a window,
the drafts verified, and the rejected ones' pages taken back by the next step;
eager, and captured once and replayed."""
import numpy as np
import pytest
import torch

from oracle import step as ref

pytestmark = pytest.mark.gpu

V, D, HQ, HKV, P = 211, 64, 4, 2, 16
WINDOW, SINKS, EPS, TEMP = 40, 3, 1e-6, 0.9


class Server:
    """Rows of tokens; queries, keys, values and logits are tables by token, so that a
    row's cache can be made again from its tokens alone."""

    def __init__(self, rows, k, q8, dt):
        gen = torch.Generator(device="cuda").manual_seed(1)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        B, n = len(rows), 1 + k
        self.B, self.n, self.dt, self.q8 = B, n, dt, q8
        self.packed = rnd(V, HQ + 2 * HKV, D).to(dt)
        self.wq, self.wk = (1 + 0.1 * rnd(D)).to(dt), (1 + 0.1 * rnd(D)).to(dt)
        self.logit = (2 * rnd(V, V)).to(dt)
        self.read = 0.1 * rnd(HQ * D, V)
        n_pages, width = B * 16, 12
        self.kc, self.vc = (torch.zeros(n_pages, HKV, P, D, dtype=torch.uint8 if q8 else dt, device="cuda") for _ in range(2))
        self.scales = {}
        if q8:
            self.scales = {x: torch.zeros(n_pages, HKV, P, 1, dtype=dt, device="cuda")
                           for x in ("k_scales", "k_biases", "v_scales", "v_biases")}
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        from gmlx_amd import ops
        self.freqs, self.factor = ops.rope_frequencies(D, scaling=dict(type="yarn", factor=4, original=64))
        self.table, self.free, self.count = i32(B, width), torch.arange(n_pages, device="cuda").int(), i32(1) + n_pages
        self.seq, self.keep, self.new = i32(B), i32(B), i32(B) + n
        self.tokens, self.u, self.draws = i32(B * n), torch.zeros(B * n, device="cuda"), torch.zeros(B, device="cuda")
        # the prompts, in one step of their own
        p = ops.paged_plan(self.seq, torch.tensor([len(r) for r in rows], device="cuda").int(), self.table, self.free,
                           self.count, P, sum(len(r) for r in rows))
        x = self.packed[torch.tensor([t for r in rows for t in r], device="cuda")]
        ops.paged_write_rope(x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], self.kc, self.vc, p.slots, p.positions,
                             self.freqs, **self.turn(), **self.scales)
        assert p.refused.sum() == 0
        self.seq.copy_(p.kv_lens)
        self.keep.copy_(p.kv_lens)
        self.count.copy_(p.free_count)

    def turn(self):
        return dict(q_weight=self.wq, k_weight=self.wk, eps=EPS, factor=self.factor)

    def step(self):
        """One step of every row on the tokens in self.tokens; the state is updated in place."""
        from gmlx_amd import ops
        T = self.B * self.n
        p = ops.paged_plan(self.seq, self.new, self.table, self.free, self.count, P, T, keep_lens=self.keep)
        x = self.packed[self.tokens.long()]
        q = ops.paged_write_rope(x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], self.kc, self.vc, p.slots, p.positions,
                                 self.freqs, **self.turn(), **self.scales)
        o = ops.sdpa_paged(q, self.kc, self.vc, self.table, p.kv_lens, p.cu_q, D ** -0.5, max_q=self.n, window=WINDOW,
                           sinks=SINKS, **self.scales)
        logits = (self.logit[self.tokens.long()].float() + o.view(T, -1).float() @ self.read).to(self.dt)
        r = ops.verify_drafts(logits, self.tokens, p.cu_q, self.u, self.draws, temperature=TEMP, kv_lens=p.kv_lens)
        self.seq.copy_(p.kv_lens)
        self.count.copy_(p.free_count)
        self.keep.copy_(r.keep_lens)
        return p, q, o, logits, r


def _next(server, last, rng):
    """Drafts that mostly follow the logits' table, and the step's random numbers."""
    n = server.n
    toks = np.zeros((server.B, n), np.int64)
    toks[:, 0] = last
    table = server.logit.float().cpu().numpy()
    for i in range(1, n):
        likely = table[toks[:, i - 1]].argmax(1)
        toks[:, i] = np.where(rng.random(server.B) < 0.8, likely, rng.integers(0, V, server.B))
    server.tokens.copy_(torch.from_numpy(toks.reshape(-1)).int())
    server.u.copy_(torch.from_numpy(rng.random(server.B * n).astype(np.float32) * 0.3))
    server.draws.copy_(torch.from_numpy(rng.random(server.B).astype(np.float32)))
    return toks


@pytest.mark.parametrize("q8,dt", [(False, torch.float16), (False, torch.bfloat16), (True, torch.bfloat16)])
def test_steps(q8, dt):
    from gmlx_amd import ops
    rng = np.random.default_rng(3)
    rows = [rng.integers(0, V, m).tolist() for m in (5, 37, 64, 1, 90)]
    eager, graph = Server(rows, 3, q8, dt), Server(rows, 3, q8, dt)
    half = torch.finfo(dt).eps / 2
    # captured on a copy of the state's numbers, which the capture's warm-up leaves changed
    held = [x.clone() for x in (graph.table, graph.free, graph.count, graph.seq, graph.keep)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph.step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = graph.step()
    torch.cuda.current_stream().wait_stream(s)
    for x, y in zip((graph.table, graph.free, graph.count, graph.seq, graph.keep), held):
        x.copy_(y)
    last = rng.integers(0, V, 5)
    stood = fell = 0
    for step in range(8):
        state = rng.bit_generator.state
        toks = _next(eager, last, rng)
        rng.bit_generator.state = state
        _next(graph, last, rng)
        p, q, o, logits, r = eager.step()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*p, q, o, logits, *r), (*out[0], *out[1:4], *out[4])):
            assert torch.equal(a, b), step
        assert p.refused.sum() == 0
        kv, acc = p.kv_lens.tolist(), r.accepted.tolist()
        for b in range(5):
            rows[b] = rows[b] + toks[b].tolist()
            assert kv[b] == len(rows[b])
            at = slice(4 * b, 4 * b + 4)
            assert p.positions[at].tolist() == list(range(kv[b] - 4, kv[b]))
            # the row's cache, made again from its tokens
            x = eager.packed[torch.tensor(rows[b], device="cuda")]
            pos = torch.arange(kv[b], dtype=torch.int32, device="cuda")
            qr, kr = ops.rope_qk(x[:, :HQ], x[:, HQ:HQ + HKV], pos, eager.freqs, **eager.turn())
            assert torch.equal(q[at], qr[-4:])
            slots = (eager.table[b, (pos // P).long()] * P + pos % P).int()
            ck, cv = ops.paged_read(eager.kc, eager.vc, slots, **eager.scales)
            if not q8:
                assert torch.equal(ck, kr) and torch.equal(cv, x[:, HQ + HKV:])
            else:
                # within half a step of the group, 1/255 of its range, and the 16-bit roundings of
                # scale (255 times half a step of it), bias and result
                for c, w in ((ck, kr), (cv, x[:, HQ + HKV:])):
                    w = w.double()
                    lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
                    assert ((c.double() - w).abs() <= (hi - lo) * (0.51 / 255 + half) + half * w.abs() + half * (hi - lo)).all()
            kd, vd = (y.double().cpu().numpy().transpose(1, 0, 2) for y in (ck, cv))
            want, far = ref.window_attention(q[at].double().cpu().numpy(), kd, vd, 4, D ** -0.5, WINDOW, SINKS)
            got = o[at].double().cpu().numpy()
            # the output's and the probabilities' roundings, 8-bit values' on top where they were read back in
            # 16 bits (keys: 64 products of up to 4 standard deviations each, in the scores), and 2^-16 for fp32
            room = half * (np.abs(want) + 1.01 * far) + 2.0 ** -16 * far + 1e-6
            if q8:
                size = np.abs(q[at].double().cpu().numpy()).sum(-1, keepdims=True) * np.abs(kd).max() * D ** -0.5
                room = room + half * far * (2 + 2 * size)
            assert (np.abs(got - want) <= room).all()
            a, t, keep = ref.verify(logits[at].double().cpu().numpy(), toks[b], [0, 4], eager.u[at].cpu().numpy(),
                                    [float(eager.draws[b])], None, TEMP, [kv[b]])
            assert (a[0], t[0], keep[0]) == (acc[b], int(r.tokens[b]), int(r.keep_lens[b]))
            rows[b] = rows[b][:keep[0]]
            stood += acc[b]
            fell += acc[b] < 3
        last = r.tokens.cpu().numpy()
    assert stood > 10 and fell > 5  # both happened
    # every page is a row's or on the stack, once
    used = [int(eager.table[b, i]) for b in range(5) for i in range(-(-int(eager.seq[b]) // P))]
    free = eager.free[:int(eager.count)].tolist()
    assert sorted(used + free) == list(range(5 * 16))


@pytest.mark.parametrize("sinks", [0, 3, 40])
def test_pages_behind_the_window_given_back_and_rows_ended(sinks):
    """Pages that no later token sees go on the stack by hand between two plans, and their rows are ended in two steps:
    what lies from the first page held behind them on by the plan, the sinks' pages by hand.  Outputs are those of a
    cache that holds everything, in a pool too small for that, and no page is ever in two places."""
    from gmlx_amd import ops
    B, n, steps, width = 3, 20, 40, 64
    rng = np.random.default_rng(sinks)
    gen = torch.Generator(device="cuda").manual_seed(sinks)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    class Cache:
        def __init__(self, n_pages):
            self.n = n_pages
            self.k, self.v = (torch.full((n_pages, HKV, P, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
            self.table, self.free, self.count = i32([[-1] * width] * B), i32(list(range(n_pages))), i32([n_pages])
            self.seq, self.hole = i32([0] * B), [(0, 0)] * B

        def step(self, new, keep, q, k, v):
            p = ops.paged_plan(self.seq, i32(new), self.table, self.free, self.count, P, sum(new), keep_lens=i32(keep))
            ops.paged_write(k, v, self.k, self.v, p.slots)
            self.seq.copy_(p.kv_lens)
            self.count.copy_(p.free_count)
            assert p.refused.sum() == 0
            return ops.sdpa_paged(q, self.k, self.v, self.table, p.kv_lens, p.cu_q, D ** -0.5, max_q=max(new), window=WINDOW,
                                  sinks=sinks)

        def push(self, b, pages):
            c = int(self.count)
            for j in pages:
                self.free[c], c = int(self.table[b, j]), c + 1
                self.table[b, j] = -1
            self.count.fill_(c)

        def give_back(self, b, kept):
            """Pages between the sinks and the window of the next new token, at position `kept`."""
            first, end = self.hole[b][1] or -(-sinks // P), max(kept + 1 - WINDOW, 0) // P
            if end > first:
                self.push(b, range(first, end))
                self.hole[b] = (-(-sinks // P), end)

        def held(self):
            return [int(x) for b in range(B) for x in self.table[b, :-(-int(self.seq[b]) // P)] if x >= 0]

        def whole(self):
            assert sorted(self.held() + self.free[:int(self.count)].tolist()) == list(range(self.n))

    # a row holds the sinks', the window's and the new tokens' pages, and what the last one had
    small, large = Cache(B * (-(-sinks // P) + (WINDOW + 2 * n) // P + 3)), Cache(B * width)
    kept, most = [0] * B, 0
    for step in range(steps):
        new = rng.integers(1, n + 1, B).tolist()
        if step % 13 == 12:
            b = step // 13 % B  # the row ends, and a new request takes its place
            if small.hole[b][1]:
                keep = [small.hole[b][1] * P if i == b else kept[i] for i in range(B)]
                assert keep[b] <= int(small.seq[b])
                p = ops.paged_plan(small.seq, i32([0] * B), small.table, small.free, small.count, P, 0, keep_lens=i32(keep))
                small.seq.copy_(p.kv_lens)
                small.count.copy_(p.free_count)
                small.push(b, range(small.hole[b][0]))
                small.seq[b], small.hole[b] = 0, (0, 0)
                small.whole()
            kept[b] = 0
        x = torch.randn(sum(new), HQ + 2 * HKV, D, device="cuda", generator=gen).half()
        a, b = (c.step(new, kept, x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]) for c in (small, large))
        assert torch.equal(a, b), step
        assert not a.isnan().any()
        small.whole()
        large.whole()
        most = max(most, len(large.held()))
        kept = [max(k, k + m - int(r)) for k, m, r in zip(kept, new, rng.integers(0, 3, B))]  # some drafts fall
        for r in range(B):
            small.give_back(r, kept[r])
    assert most > small.n


def test_a_row_that_the_plan_refuses_keeps_what_it_kept():
    """A row without pages for its new tokens stays as it was, with the drafts of the step before still at its end: its
    verdict is of no use, and what it keeps is what it kept.  It goes on when pages come free, its cache whole."""
    from gmlx_amd import ops
    dt, n, width = torch.float16, 4, 8
    rng = np.random.default_rng(5)
    gen = torch.Generator(device="cuda").manual_seed(5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    packed = torch.randn(V, HQ + 2 * HKV, D, device="cuda", generator=gen).to(dt)
    freqs, _ = ops.rope_frequencies(D)
    n_pages = 7
    kc, vc = (torch.zeros(n_pages, HKV, P, D, dtype=dt, device="cuda") for _ in range(2))
    table, free, count = i32([[-1] * width] * 3), i32(list(range(n_pages))), i32([n_pages])
    rows = [rng.integers(0, V, m).tolist() for m in (30, 20, 40)]
    seq, kept = i32([0, 0, 0]), i32([0, 0, 0])

    def step(new, toks):
        p = ops.paged_plan(seq, i32(new), table, free, count, P, len(toks), keep_lens=kept)
        x = packed[torch.tensor(toks, device="cuda")]
        ops.paged_write_rope(x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], kc, vc, p.slots, p.positions, freqs)
        seq.copy_(p.kv_lens)
        count.copy_(p.free_count)
        return p
    p = step([30, 20, 40], sum(rows, []))  # 2 + 2 + 3 pages: none left
    assert p.refused.sum() == 0 and int(p.free_count) == 0
    kept.copy_(p.kv_lens)
    refusals = went_on = 0
    for t in range(12):
        if t == 7:  # the third row ends
            kept[2], rows[2] = 0, []
        toks = [rng.integers(0, V, n).tolist() for _ in range(3)]
        before = kept.tolist()
        assert before == [len(r) for r in rows]
        p = step([n, n, n if t < 7 else 0], sum(toks[:3 if t < 7 else 2], []))
        T = 3 * n if t < 7 else 2 * n
        logits = torch.randn(T, V, device="cuda", generator=gen)
        r = ops.verify_drafts(logits, i32(sum(toks, [])[:T]), p.cu_q, torch.rand(T, device="cuda", generator=gen) * 0.02,
                              torch.rand(3, device="cuda", generator=gen), kv_lens=p.kv_lens)
        # a row without new tokens keeps all, a refused one what it kept
        kept.copy_(torch.where(p.refused > 0, kept, r.keep_lens))
        for b in range(3):
            if p.refused[b]:
                refusals += 1
                assert int(kept[b]) == before[b] <= int(seq[b]) == int(p.kv_lens[b])
            elif t < 7 or b < 2:
                rows[b] = (rows[b] + toks[b])[:int(kept[b])]
                assert len(rows[b]) == int(kept[b]) == before[b] + 1 + int(r.accepted[b])
                went_on += t > 7 and refusals > 0
            pos = torch.arange(len(rows[b]), dtype=torch.int32, device="cuda")
            if len(pos):
                x = packed[torch.tensor(rows[b], device="cuda")]
                _, kr = ops.rope_qk(x[:, :HQ], x[:, HQ:HQ + HKV], pos, freqs)
                ck, cv = ops.paged_read(kc, vc, (table[b, (pos // P).long()] * P + pos % P).int())
                assert torch.equal(ck, kr) and torch.equal(cv, x[:, HQ + HKV:]), (t, b)
    assert refusals > 3 and went_on > 3
