"""Host side of the operators around a paged step: refusals of the C ABI before any
launch, the frequencies, and the references' own invariants.  No GPU needed."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import step as ref


def _lib():
    from gmlx_amd import _lib as m
    return m, m.lib()


X = 1 << 26


def _rope(m, **kw):
    d = dict(freqs=X, q_weight=None, k_weight=None, weight_dtype=m.DTYPE_F16, rotary_dim=128, interleaved=0, eps=1e-6,
             factor=1.0)
    d.update(kw)
    return ctypes.byref(m.Rope(*d.values()))


def _rows(m, **kw):
    d = dict(x=X, out=X, token_stride=1024, head_stride=128, out_token_stride=1024, out_head_stride=128, heads=8)
    d.update(kw)
    return ctypes.byref(m.RopeRows(*d.values()))


def _pool(m, **kw):
    d = dict(k=1 << 20, v=1 << 21, k_scales=None, k_biases=None, v_scales=None, v_biases=None, page_stride=8 * 16 * 128,
             head_stride=16 * 128, token_stride=128, n_pages=10, page_size=16, Hkv=8, D=128, dtype=m.DTYPE_F16)
    d.update(kw)
    return ctypes.byref(m.PagedPool(**d))


def test_rope_calls_are_refused():
    m, L = _lib()

    def call(rope=None, pos=X, T=4, D=128, dt=m.DTYPE_F16, q=None, k=None):
        return L.kq_rope_qk(rope or _rope(m), pos, T, D, dt, q or _rows(m), k or _rows(m), None)

    def write(pool=None, rope=None, pos=X, slots=X, T=4, q=None, k=X, kt=1024, v=X, vh=128):
        return L.kq_paged_write_rope(pool or _pool(m), rope or _rope(m), pos, slots, T, q or _rows(m), k, kt, 128, v, 1024, vh,
                                     None)
    assert call(T=0) == m.KQ_OK and write(T=0) == m.KQ_OK
    for bad, code in ((dict(freqs=None), "NULL_POINTER"), (dict(rotary_dim=0), "BAD_SHAPE"),
                      (dict(rotary_dim=24), "BAD_SHAPE"), (dict(rotary_dim=144), "BAD_SHAPE"),
                      (dict(q_weight=X, weight_dtype=m.DTYPE_BF16), "UNSUPPORTED_DTYPE"),
                      (dict(eps=-1.0), "BAD_ARGUMENT"), (dict(eps=math.nan), "BAD_ARGUMENT"),
                      (dict(factor=math.inf), "BAD_ARGUMENT"), (dict(factor=math.nan), "BAD_ARGUMENT"),
                      (dict(freqs=X + 4), "BAD_ALIGN"), (dict(k_weight=X + 8), "BAD_ALIGN")):
        want = getattr(m, "KQ_ERR_" + code)
        assert call(rope=_rope(m, **bad)) == want and write(rope=_rope(m, **bad)) == want, bad
    for bad, code in ((dict(x=None), "NULL_POINTER"), (dict(out=None), "NULL_POINTER"), (dict(x=X + 8), "BAD_ALIGN"),
                      (dict(out=X + 2), "BAD_ALIGN"), (dict(token_stride=1025), "BAD_ALIGN"),
                      (dict(out_head_stride=4), "BAD_ALIGN"), (dict(heads=-1), "BAD_SHAPE"),
                      (dict(heads=(1 << 16) + 1), "BAD_SHAPE")):
        want = getattr(m, "KQ_ERR_" + code)
        assert call(q=_rows(m, **bad)) == want and call(k=_rows(m, **bad)) == want and write(q=_rows(m, **bad)) == want, bad
    for bad, code in ((dict(pos=None), "NULL_POINTER"), (dict(T=-1), "BAD_SHAPE"), (dict(T=(1 << 23) + 1), "BAD_SHAPE"),
                      (dict(D=80), "BAD_SHAPE"), (dict(dt=m.DTYPE_F32), "UNSUPPORTED_DTYPE")):
        assert call(**bad) == getattr(m, "KQ_ERR_" + code), bad
    for bad, code in ((dict(pool=_pool(m, D=80)), "BAD_SHAPE"), (dict(pool=_pool(m, page_stride=0)), "BAD_ARGUMENT"),
                      (dict(slots=None), "NULL_POINTER"), (dict(k=None), "NULL_POINTER"), (dict(v=None), "NULL_POINTER"),
                      (dict(v=X + 2), "BAD_ALIGN"), (dict(kt=1020), "BAD_ALIGN"), (dict(vh=12), "BAD_ALIGN"),
                      (dict(T=-1), "BAD_SHAPE")):
        assert write(**bad) == getattr(m, "KQ_ERR_" + code), bad
    none = _rows(m, x=None, out=None, heads=0)
    assert call(q=none, k=none) == m.KQ_OK  # no heads: nothing to do


def test_outputs_at_an_inputs_address():
    """Strides of a dimension of one say nothing of where its rows lie."""
    from gmlx_amd import ops
    buf = torch.zeros(6 * 12 * 64, dtype=torch.float16)
    at = lambda T, H, t, h: buf.as_strided((T, H, 64), (t, h, 1))  # noqa: E731
    for x, out in ((at(1, 8, 768, 64), at(1, 8, 512, 64)), (at(5, 1, 768, 64), at(5, 1, 768, 768)),
                   (at(1, 1, 768, 64), at(1, 1, 64, 768)), (at(5, 8, 768, 64), at(5, 8, 768, 64)),
                   (at(0, 8, 768, 64), at(0, 8, 512, 128))):
        assert ops._rope_rows("rope_qk", "q", x, out)[1] is out
    for x, out in ((at(2, 8, 768, 64), at(2, 8, 512, 64)), (at(1, 5, 768, 64), at(1, 5, 768, 128)),
                   (at(5, 8, 768, 64), at(5, 8, 64, 320))):
        with pytest.raises(ValueError):
            ops._rope_rows("rope_qk", "q", x, out)


def test_verify_calls_are_refused():
    m, L = _lib()

    def call(**kw):
        d = dict(x=X, dt=m.DTYPE_F16, stride=100, tok=X, cu=X, u=X, r=X, p=None, pt=0, ps=0, temps=None, temp=1.0, kv=X, T=4,
                 B=2, V=100, acc=X, nxt=X, keep=X, ws=X, n=1 << 20)
        d.update(kw)
        return L.kq_verify_drafts(*d.values(), None)
    assert call(B=0) == m.KQ_OK
    for name in ("x", "tok", "cu", "u", "r", "kv", "acc", "nxt"):
        assert call(**{name: None}) == m.KQ_ERR_NULL_POINTER, name
    for bad in (dict(T=-1), dict(B=-1), dict(V=0), dict(stride=-1), dict(B=1 << 16), dict(T=(1 << 22) + 1),
                dict(V=(1 << 28) + 1), dict(T=1 << 20, V=1 << 20), dict(p=X, pt=0, ps=-1)):
        assert call(**bad) == m.KQ_ERR_BAD_SHAPE, bad
    for bad in (dict(dt=3), dict(dt=-1), dict(p=X, pt=7)):
        assert call(**bad) == m.KQ_ERR_UNSUPPORTED_DTYPE, bad
    for bad in (dict(temp=-1.0), dict(temp=math.nan), dict(temp=math.inf)):
        assert call(**bad) == m.KQ_ERR_BAD_ARGUMENT, bad
    for bad in (dict(x=X + 1), dict(x=X + 2, dt=m.DTYPE_F32), dict(p=X + 2, pt=m.DTYPE_F32), dict(ws=X + 128)):
        assert call(**bad) == m.KQ_ERR_BAD_ALIGN, bad
    need = L.kq_verify_workspace_bytes(4, 2, 100, m.DTYPE_F16, 1)
    assert need > L.kq_verify_workspace_bytes(4, 2, 100, m.DTYPE_F16, 0) > 0
    assert call(ws=None) == m.KQ_ERR_WORKSPACE_TOO_SMALL
    assert call(p=X, pt=m.DTYPE_F32, ps=100, n=need - 1) == m.KQ_ERR_WORKSPACE_TOO_SMALL
    for bad in ((0, 2, 100, 1), (4, 0, 100, 1), (4, 2, 0, 1), (4, 2, 100, 9), (1 << 20, 2, 1 << 20, 1)):
        assert L.kq_verify_workspace_bytes(*bad, 1) == 0, bad


def test_a_temperature_crosses_the_c_abi_in_64_bits():
    m, L = _lib()
    args = dict(x=X, dt=m.DTYPE_F16, stride=100, tok=X, cu=X, u=None, r=None, p=None, pt=0, ps=0, temps=None, temp=0.0, kv=X,
                T=4, B=2, V=100, acc=X, nxt=X, keep=X, ws=None, n=0)
    call = lambda temp: L.kq_verify_drafts(*{**args, "temp": temp}.values(), None)  # noqa: E731
    # 0 needs no random numbers; one that 32 bits would round to 0 or to infinity is as any other
    assert call(0.0) == m.KQ_ERR_WORKSPACE_TOO_SMALL
    for temp in (1e-60, 0.7, 1e60):
        assert call(temp) == m.KQ_ERR_NULL_POINTER, temp


def test_frequencies():
    from gmlx_amd import ops
    f, by = ops.rope_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and by == 1.0
    assert torch.allclose(f, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14, atol=0)
    lin, _ = ops.rope_frequencies(64, 10000.0, dict(type="linear", factor=4), device="cpu")
    assert torch.allclose(lin, f / 4, rtol=1e-14, atol=0)
    ntk, _ = ops.rope_frequencies(64, 10000.0, dict(type="ntk", factor=4), device="cpu")
    assert ntk[0] == 1 and abs(ntk[-1] / (f[-1] / 4) - 1) < 1e-12
    bands, by = ops.rope_frequencies(64, 10000.0, dict(type="bands", factor=8, original=8192), device="cpu")
    turns = 8192 * f / (2 * math.pi)
    assert by == 1.0 and torch.equal(bands[turns > 4], f[turns > 4])
    assert torch.allclose(bands[turns < 1], f[turns < 1] / 8, rtol=1e-14, atol=0)
    mid = (turns >= 1) & (turns <= 4)
    assert mid.any() and ((bands[mid] <= f[mid]) & (bands[mid] >= f[mid] / 8)).all()
    yarn, by = ops.rope_frequencies(64, 10000.0, dict(type="yarn", factor=16, original=4096), device="cpu")
    assert abs(by - (0.1 * math.log(16) + 1)) < 1e-15
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 32.0 * 10000 ** (1 / 32)], f[turns > 32.0 * 10000 ** (1 / 32)])
    slow = turns < 10000.0 ** (-1 / 32)
    assert torch.allclose(yarn[slow], f[slow] / 16, rtol=1e-14, atol=0)
    assert ops.rope_frequencies(64, scaling=dict(type="yarn", factor=2, original=64, attention=1.5), device="cpu")[1] == 1.5
    for bad in (dict(type="other"), dict(type="linear", factor=0.5), dict(type="bands", factor=2),
                dict(type="yarn", factor=2, original=100, low=4, high=2), dict(type="linear", factor=math.inf)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(64, scaling=bad, device="cpu")
    for R, base in ((0, 1e4), (7, 1e4), (64, 1.0), (64, math.inf), (64, math.nan)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(R, base, device="cpu")


def test_rope_reference_keeps_lengths_and_differences():
    """A rotation keeps a row's length, and the product of two rows goes by the
    distance of their positions alone."""
    rng = np.random.default_rng(1)
    q, k = rng.normal(size=(2, 1, 1, 64))
    f = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    for inter in (False, True):
        a, _ = ref.rope(q, [100], f, interleaved=inter)
        b, _ = ref.rope(k, [93], f, interleaved=inter)
        c, _ = ref.rope(q, [7], f, interleaved=inter)
        assert abs((a * a).sum() - (q * q).sum()) < 1e-10
        assert abs((a * b).sum() - (c * k).sum()) < 1e-10


def test_verify_reference():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.2, 0.7], [0.6, 0.2, 0.2]]))
    # both stand, then the last row's draw
    assert ref.verify_row(x, [0, 2], [0.4, 0.6, 0], 0.7, None, 1.0) == (2, 1)
    # the second falls: drawn from the others, 0.1 : 0.2
    assert ref.verify_row(x, [0, 2], [0.4, 0.75, 0], 0.2, None, 1.0) == (1, 0)
    assert ref.verify_row(x, [0, 2], [0.4, 0.75, 0], 0.5, None, 1.0) == (1, 1)
    # beside q: max(p - q, 0) is token 2's alone
    assert ref.verify_row(x[1:], [1], [0.5, 0], 0.3, np.array([[0.1, 0.6, 0.3]] * 2), 1.0) == (0, 2)
    assert ref.verify_row(x, [0, 2], [0, 0, 0], 0, None, 0.0) == (2, 0)
    assert ref.verify_row(x, [1, 2], [0, 0, 0], 0, None, 0.0) == (0, 0)
    assert ref.verify_row(x[:0], [], [], 0.5, None, 1.0) == (0, -1)


def test_window_calls_are_refused_and_sized():
    m, L = _lib()
    pool = _pool(m)

    def call(window=64, sinks=4, **kw):
        d = dict(T=4, B=2, Hq=32, mq=4, mkv=64, q=X, ws=None, n=0)
        d.update(kw)
        return L.kq_sdpa_paged_window(d["q"], 4096, pool, X, 4, 4, X, X, d["T"], d["B"], d["Hq"], d["mq"], d["mkv"], window,
                                      sinks, 0.1, X, 4096, d["ws"], d["n"], None)
    for bad in (dict(window=0), dict(window=-1), dict(window=(1 << 30) + 1), dict(sinks=-1), dict(sinks=(1 << 30) + 1),
                dict(Hq=12), dict(mq=0), dict(T=-1)):
        assert call(**bad) == m.KQ_ERR_BAD_SHAPE, bad
    assert call(q=None) == m.KQ_ERR_NULL_POINTER and call(T=0) == m.KQ_OK
    size = lambda mkv, w, s, mq=4: L.kq_sdpa_paged_window_workspace_bytes(4, 2, 32, 8, 128, mq, mkv, 0, w, s)  # noqa: E731
    whole = L.kq_sdpa_paged_workspace_bytes(4, 2, 32, 8, 128, 4, 1 << 20, 0)
    # by the window, not the rows: the same at any length, and never more than without
    assert 0 < size(1 << 20, 4096, 4) == size(1 << 30, 4096, 4) < whole
    assert size(1 << 20, 1 << 30, 0) == size(1 << 20, 64, 1 << 30) == whole
    assert size(1 << 20, 0, 0) == size(1 << 20, 4, -1) == 0
    assert call(window=4096, mkv=1 << 20) == m.KQ_ERR_WORKSPACE_TOO_SMALL


@pytest.mark.parametrize("Hq,Hkv,D,q8", [(32, 8, 128, 0), (32, 8, 128, 1), (64, 4, 128, 0), (16, 2, 256, 0), (16, 2, 256, 1)])
def test_a_window_far_past_the_rows_keeps_their_splits(Hq, Hkv, D, q8):
    """The workspace counts a call's splits: those of the rows, not of a window that none of them fills."""
    L = _lib()[1]
    for keys in (1600, 2000, 6000, 8000, 12000):
        whole = L.kq_sdpa_paged_workspace_bytes(4, 4, Hq, Hkv, D, 1, keys, q8)
        for window, sinks in ((16385, 0), (16320, 65), (32768, 4), (1 << 18, 0), (1 << 30, 1 << 30), (64, 1 << 20)):
            assert L.kq_sdpa_paged_window_workspace_bytes(4, 4, Hq, Hkv, D, 1, keys, q8, window, sinks) == whole


def test_window_reference():
    rng = np.random.default_rng(2)
    q, k, v = rng.normal(size=(3, 2, 8)), rng.normal(size=(1, 20, 8)), rng.normal(size=(1, 20, 8))
    out, _ = ref.window_attention(q, k, v, 3, 0.3, 4, 2)
    # token 1 is key 18: it sees 0, 1, 15 .. 18
    see = [0, 1, 15, 16, 17, 18]
    p = np.exp(q[1, 1] @ k[0, see].T * 0.3)
    assert np.allclose(out[1, 1], p @ v[0, see] / p.sum())
