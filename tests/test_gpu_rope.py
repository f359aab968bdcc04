"""Head norms and rotations by position on the GPU, alone and into a paged cache,
against fp64 numpy and against the two calls that the joined one stands for."""
import numpy as np
import pytest
import torch

from oracle import step as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step of a rounding, relative


def _say(*a):
    print(*a, flush=True)


def _freqs(R, base=10000.0):
    from gmlx_amd import ops
    return ops.rope_frequencies(R, base)[0]


def _check(got, x, positions, freqs, weight, eps, interleaved, factor):
    """Half a step of the output, and in fp32 steps of 2^-24 of the values that
    meet in it: the norm (8 + 6 sums of squares, at half each, mean, eps, root,
    quotient and two products: 13), the turn's conversion (pi), sine, cosine and
    factor (4), products and sum (3), the angle of 64 bits at 2^31 (8): below 40."""
    want, size = ref.rope(x.double().cpu().numpy(), positions, freqs.cpu().numpy(), weight, eps, interleaved, factor)
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    d = np.abs(got.double().cpu().numpy() - want)
    room = HALF[x.dtype] * np.abs(want) + 40 * 2.0 ** -24 * size + tiny
    assert np.isfinite(d).all() and (d <= room).all(), (d / room).max()


CASES = [  # T, Hq, Hkv, D, R, interleaved, norm
    (1, 32, 8, 128, 128, False, True), (3, 4, 1, 64, 64, True, True), (7, 12, 3, 96, 48, False, True),
    (5, 3, 1, 96, 96, True, False), (33, 16, 2, 256, 64, False, True), (2, 5, 5, 512, 512, False, True),
    (9, 8, 1, 512, 16, True, True), (130, 7, 2, 128, 112, False, False), (515, 6, 2, 128, 128, False, True),
    (777, 9, 4, 64, 32, True, True), (600, 4, 2, 256, 256, True, True), (513, 3, 1, 512, 256, False, True),
    (514, 20, 4, 96, 96, False, True),
    # several tokens a workgroup: a last one of few, a lone head, one token too many for the passes
    (9001, 2, 1, 64, 64, False, True), (7003, 1, 0, 128, 128, True, True), (4099, 5, 1, 256, 128, False, False),
    (3085, 2, 1, 512, 512, False, True), (4100, 7, 1, 96, 64, True, True), (4111, 16, 8, 128, 128, False, True)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,interleaved,norm", CASES)
def test_rope(T, Hq, Hkv, D, R, interleaved, norm, dt):
    from gmlx_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(T * D + Hq)
    packed = torch.randn(T, Hq + 2 * Hkv, D, device="cuda", generator=gen).to(dt)
    q, k = packed[:, :Hq], packed[:, Hq:Hq + Hkv]
    pos = torch.randint(0, 100000, (T,), device="cuda", generator=gen, dtype=torch.int32)
    pos[0] = 0
    wt = torch.float32 if D == 64 else dt
    wq, wk = ((1 + torch.randn(D, device="cuda", generator=gen)).to(wt) for _ in range(2))
    freqs = _freqs(R)
    kw = dict(interleaved=interleaved, factor=1.25 if R < D else 1.0)
    if norm:
        kw.update(q_weight=wq, k_weight=wk, eps=1e-5)
    _say("rope", T, Hq, Hkv, D, R, interleaved, norm, dt)
    gq, gk = ops.rope_qk(q, k, pos, freqs, **kw)
    for got, x, w in ((gq, q, wq), (gk, k, wk)):
        _check(got, x, pos.cpu().numpy(), freqs, w.double().cpu().numpy() if norm else None, 1e-5, interleaved, kw["factor"])
    # a row alone has the same bits, and so has the call in place
    i = T // 2
    oq, ok = ops.rope_qk(q[i:i + 1], k[i:i + 1], pos[i:i + 1], freqs, **kw)
    assert torch.equal(oq[0], gq[i]) and torch.equal(ok[0], gk[i])
    iq, ik = ops.rope_qk(q, k, pos, freqs, q_out=q, k_out=k, **kw)
    assert iq.data_ptr() == packed.data_ptr() and torch.equal(q, gq) and torch.equal(k, gk)


def test_far_positions_and_a_norm_on_one_side():
    from gmlx_amd import ops
    torch.manual_seed(1)
    pos = torch.tensor([0, 1, 131071, 10 ** 6, 16777217, 2 ** 30 + 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    for dt in (F16, BF16):
        q, k = torch.randn(7, 3, 128, device="cuda").to(dt), torch.randn(7, 2, 128, device="cuda").to(dt)
        w = torch.randn(128, device="cuda").to(dt)
        freqs = _freqs(128, 1e6)
        _say("far", dt)
        gq, gk = ops.rope_qk(q, k, pos, freqs, k_weight=w)
        _check(gq, q, pos.cpu().numpy(), freqs, None, 0, False, 1.0)
        _check(gk, k, pos.cpu().numpy(), freqs, w.double().cpu().numpy(), 1e-6, False, 1.0)


def test_tokens_without_a_position_stay():
    from gmlx_amd import ops
    q, k = torch.randn(6, 4, 64, device="cuda").half(), torch.randn(6, 2, 64, device="cuda").half()
    pos = torch.tensor([5, -1, 7, -2 ** 31, 0, -1], dtype=torch.int32, device="cuda")
    qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    freqs = _freqs(64)
    ops.rope_qk(q, k, pos, freqs, q_out=qo, k_out=ko)
    full = ops.rope_qk(q, k, pos.clamp(min=0), freqs)
    for got, want in ((qo, full[0]), (ko, full[1])):
        for t, p in enumerate(pos.tolist()):
            assert torch.equal(got[t], want[t]) if p >= 0 else (got[t] == 9).all()


def test_values_past_the_root_of_the_largest():
    """bf16 rows whose squares pass fp32, tiny ones, and infinities and NaN, which
    stay in their rows."""
    from gmlx_amd import ops
    torch.manual_seed(2)
    q = torch.randn(8, 2, 128, device="cuda")
    q[0] *= 1e37
    q[1] *= 1e30
    q[2] *= 1e-30
    q[3] *= 1e19
    q = q.clamp(-3.3e38, 3.3e38).to(BF16)
    k = torch.randn(8, 1, 128, device="cuda").to(BF16)
    w = torch.randn(128, device="cuda").to(BF16)
    pos = torch.arange(8, dtype=torch.int32, device="cuda") * 1000
    freqs = _freqs(128)
    got, _ = ops.rope_qk(q, k, pos, freqs, q_weight=w, k_weight=w)
    _check(got, q, pos.cpu().numpy(), freqs, w.double().cpu().numpy(), 1e-6, False, 1.0)
    bad = q.clone()
    bad[4, 0, 3], bad[5, 1, 100] = float("nan"), float("inf")
    odd, _ = ops.rope_qk(bad, k, pos, freqs, q_weight=w, k_weight=w)
    assert torch.isnan(odd[4, 0]).all() and not torch.isfinite(odd[5, 1]).all()
    hit = torch.zeros(8, 2, dtype=torch.bool, device="cuda")
    hit[4, 0] = hit[5, 1] = True
    assert torch.equal(odd[~hit], got[~hit])
    # without a norm an infinity meets its pair alone
    plain, _ = ops.rope_qk(bad, k, pos, freqs)
    assert torch.isfinite(plain[5, 1][[i for i in range(128) if i not in (36, 100)]].float()).all()


def _pool(n, H, P, D, dt, q8, token_layout):
    def make(width, dtype):
        if token_layout:
            return [torch.zeros(n, P, H, width, dtype=dtype, device="cuda").permute(0, 2, 1, 3) for _ in range(2)]
        return [torch.zeros(n, H, P, width, dtype=dtype, device="cuda") for _ in range(2)]
    if not q8:
        return make(D, dt), {}
    (ks, vs), (kb, vb) = make(D // 64, dt), make(D // 64, dt)
    return make(D, torch.uint8), dict(k_scales=ks, k_biases=kb, v_scales=vs, v_biases=vb)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,interleaved,P,q8,token_layout", [
    (1, 32, 8, 128, 128, False, 16, False, False), (37, 16, 2, 256, 64, True, 32, True, False),
    (520, 6, 3, 96, 32, False, 64, False, True), (600, 4, 1, 64, 64, False, 128, True, False),
    (19, 3, 1, 512, 512, True, 16, True, False), (700, 8, 2, 128, 128, False, 1024, True, False),
    (5, 0, 2, 128, 64, False, 16, False, False), (6500, 2, 1, 64, 64, False, 32, False, False),
    (4201, 4, 2, 128, 128, True, 16, True, False), (3077, 1, 1, 512, 256, False, 64, False, True)])
def test_write_rope_is_the_two_calls(T, Hq, Hkv, D, R, interleaved, P, q8, token_layout, dt):
    from gmlx_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(T + D)
    n = T // P + 3
    packed = torch.randn(T, Hq + 2 * Hkv, D, device="cuda", generator=gen).to(dt)
    q, k, v = packed[:, :Hq], packed[:, Hq:Hq + Hkv], packed[:, Hq + Hkv:]
    if T > 4:
        v[3, 0, 5] = float("inf")
    pos = torch.randint(0, 50000, (T,), device="cuda", generator=gen, dtype=torch.int32)
    slots = torch.randperm(n * P, device="cuda", generator=gen)[:T].int()
    if T > 10:
        slots[2], slots[7], slots[9] = -1, n * P, 2 ** 31 - 1
        pos[1], pos[4] = -1, -7
    w = [torch.randn(D, device="cuda", generator=gen).to(dt) for _ in range(2)]
    kw = dict(q_weight=w[0], k_weight=w[1], interleaved=interleaved, factor=0.75)
    freqs = _freqs(R)
    _say("write rope", T, Hq, Hkv, D, R, P, q8, dt)
    (kc, vc), sc = _pool(n, Hkv, P, D, dt, q8, token_layout)
    (kd, vd), sd = _pool(n, Hkv, P, D, dt, q8, token_layout)
    q1, q2 = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
    ops.paged_write_rope(q, k, v, kc, vc, slots, pos, freqs, q_out=q1, **kw, **sc)
    _, kr = ops.rope_qk(q, k, pos, freqs, q_out=q2, **kw)
    ops.paged_write(kr, v, kd, vd, torch.where(pos < 0, -1, slots), **sd)
    bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(bits(q1), bits(q2))
    for a, b in ((kc, kd), (vc, vd), *((sc[x], sd[x]) for x in sc)):
        assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("T", [3, 2000, 9001])
def test_write_rope_in_place(T):
    """The queries rotated where they lie, beside the keys and values that are read."""
    from gmlx_amd import ops
    torch.manual_seed(T)
    Hq, Hkv, D, P = (32, 8, 128, 16) if T < 9000 else (2, 1, 64, 16)
    packed = torch.randn(T, Hq + 2 * Hkv, D, device="cuda").half()
    q, k, v = packed[:, :Hq], packed[:, Hq:Hq + Hkv], packed[:, Hq + Hkv:]
    kv = packed[:, Hq:].clone()
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    slots, w = pos.clone(), torch.randn(D, device="cuda")
    freqs = _freqs(D)
    (a, b), _ = _pool(-(-T // P), Hkv, P, D, F16, False, True)
    (c, d), _ = _pool(-(-T // P), Hkv, P, D, F16, False, True)
    want = ops.paged_write_rope(q, k, v, a, b, slots, pos, freqs, q_weight=w, k_weight=w)
    got = ops.paged_write_rope(q, k, v, c, d, slots, pos, freqs, q_weight=w, k_weight=w, q_out=q)
    assert got is q and torch.equal(q, want) and torch.equal(a, c) and torch.equal(b, d)
    assert torch.equal(packed[:, Hq:], kv)


@pytest.mark.parametrize("T,Hq", [(1, 8), (5, 1), (1, 1)])
def test_in_place_where_a_dimension_is_one(T, Hq):
    """A view of one token, or of one head, whose stride there is another than the output's."""
    from gmlx_amd import ops
    torch.manual_seed(T)
    buf, k = torch.randn(T * Hq * 128, device="cuda").half(), torch.randn(T, 2, 128, device="cuda").half()
    at = lambda odd: buf.as_strided((T, Hq, 128), (Hq * 128 if T > 1 else odd, 128 if Hq > 1 else odd, 1))  # noqa: E731
    pos = torch.arange(T, dtype=torch.int32, device="cuda") + 7
    want = ops.rope_qk(at(128), k, pos, _freqs(128))
    out = at(4096)
    got = ops.rope_qk(at(128), k, pos, _freqs(128), q_out=out)
    assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T,Hq,Hkv,D", [(360000, 32, 8, 128), (2200000, 4, 2, 128)])
def test_rows_past_32_bits_of_values(T, Hq, Hkv, D):
    """Each token is its own: the last ones have the bits of a call on them alone, one or several tokens a workgroup."""
    from gmlx_amd import ops
    _say("long", T)
    n, P, step = 777, 256, Hq + 2 * Hkv
    assert T * step * D > 2 ** 31
    packed = torch.empty(T, step, D, dtype=F16, device="cuda")
    for c in packed.split(100000):
        c.normal_()
    q, k, v = packed[:, :Hq], packed[:, Hq:Hq + Hkv], packed[:, Hq + Hkv:]
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 3
    freqs, w = _freqs(D), torch.randn(D, device="cuda")
    pages = -(-T // P)
    slots = pos // 3
    kw = dict(q_weight=w, k_weight=w)
    last = packed[-n:].clone()
    lq, lk, lv = last[:, :Hq], last[:, Hq:Hq + Hkv], last[:, Hq + Hkv:]
    want = ops.rope_qk(lq, lk, pos[-n:].clone(), freqs, **kw)
    got = ops.rope_qk(q, k, pos, freqs, **kw)
    assert torch.equal(got[0][-n:], want[0]) and torch.equal(got[1][-n:], want[1])
    del got
    kc, vc = (torch.zeros(pages, Hkv, P, D, dtype=F16, device="cuda") for _ in range(2))
    out = ops.paged_write_rope(q, k, v, kc, vc, slots, pos, freqs, q_out=q, **kw)
    assert torch.equal(out[-n:], want[0])
    ck, cv = ops.paged_read(kc, vc, slots[-n:].clone())
    assert torch.equal(ck, want[1]) and torch.equal(cv, lv)


def test_captured_and_on_another_stream():
    from gmlx_amd import ops
    torch.manual_seed(3)
    q, k = torch.randn(9, 8, 128, device="cuda").half(), torch.randn(9, 2, 128, device="cuda").half()
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    freqs = _freqs(128)
    w = torch.randn(128, device="cuda").half()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.rope_qk(q, k, pos, freqs, q_weight=w, k_weight=w)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = ops.rope_qk(q, k, pos, freqs, q_weight=w, k_weight=w)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        pos += i
        q *= 0.5
        g.replay()
        torch.cuda.synchronize()
        want = ops.rope_qk(q, k, pos, freqs, q_weight=w, k_weight=w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert other[0].shape == q.shape


def test_refusals():
    from gmlx_amd import ops
    q, k = torch.randn(4, 8, 128, device="cuda").half(), torch.randn(4, 2, 128, device="cuda").half()
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    f, w = _freqs(128), torch.ones(128, device="cuda").half()
    for bad in (dict(q=q.float()), dict(k=k[:3]), dict(k=k.bfloat16()), dict(q=q[..., :80], k=k[..., :80]), dict(q=q[0]),
                dict(pos=pos[:3]), dict(pos=pos.long()), dict(f=f.float()), dict(f=f[:5]), dict(f=f.cpu()),
                dict(f=torch.cat([f, f])), dict(f=f[::2]), dict(q_weight=w[:64]), dict(q_weight=w.bfloat16()),
                dict(q_weight=w, k_weight=w.float()), dict(eps=-1.0), dict(eps=float("nan")), dict(factor=float("inf")),
                dict(q_out=q[:3]), dict(q_out=k), dict(k_out=torch.empty(4, 2, 256, device="cuda").half()[..., ::2]),
                dict(k_out=torch.empty(1, 2, 128, device="cuda").half().expand(4, 2, 128)),
                dict(q_out=torch.empty(4 * 8 * 128 + 1, device="cuda").half()[1:].view(4, 8, 128))):
        d = dict(q=q, k=k, pos=pos, f=f)
        d.update({x: y for x, y in bad.items() if x in d})
        kw = {x: y for x, y in bad.items() if x not in d}
        with pytest.raises(ValueError):
            ops.rope_qk(d["q"], d["k"], d["pos"], d["f"], **kw)
    empty = ops.rope_qk(q[:0], k[:0], pos[:0], f)
    assert empty[0].shape == (0, 8, 128) and empty[1].shape == (0, 2, 128)
