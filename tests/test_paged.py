"""The paged cache's host side: refusals of the C ABI and of the ops, workspace
sizes, and the plan reference's own invariants.  No GPU needed."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import paged as ref


def _lib():
    from gmlx_amd import _lib as m
    return m, m.lib()


def _pool(**kw):
    m, _ = _lib()
    d = dict(k=1 << 20, v=1 << 21, k_scales=None, k_biases=None, v_scales=None, v_biases=None, page_stride=8 * 16 * 128,
             head_stride=16 * 128, token_stride=128, n_pages=10, page_size=16, Hkv=8, D=128, dtype=m.DTYPE_F16)
    d.update(kw)
    return m.PagedPool(**d)


Q8 = dict(k_scales=1 << 22, k_biases=1 << 23, v_scales=1 << 24, v_biases=1 << 25)


@pytest.mark.parametrize("change,code", [
    (dict(k=None), "NULL_POINTER"), (dict(v=None), "NULL_POINTER"), (dict(dtype=0), "UNSUPPORTED_DTYPE"),
    (dict(D=80), "BAD_SHAPE"), (dict(D=0), "BAD_SHAPE"), (dict(n_pages=0), "BAD_SHAPE"), (dict(Hkv=0), "BAD_SHAPE"),
    (dict(page_size=8), "BAD_SHAPE"), (dict(page_size=48), "BAD_SHAPE"), (dict(page_size=2048), "BAD_SHAPE"),
    (dict(n_pages=1 << 27), "BAD_SHAPE"), (dict(token_stride=64), "BAD_SHAPE"), (dict(token_stride=1 << 21), "BAD_SHAPE"),
    (dict(page_stride=-8), "BAD_SHAPE"), (dict(k=(1 << 20) + 8), "BAD_ALIGN"), (dict(head_stride=2052), "BAD_ALIGN"),
    (dict(**{**Q8, "v_biases": None}), "NULL_POINTER"), (dict(**Q8, D=96, token_stride=96), "BAD_ALIGN"),
    (dict(**Q8, D=96, token_stride=128), "BAD_SHAPE"),
    (dict(**Q8, token_stride=1024), "BAD_SHAPE"), (dict(**Q8, head_stride=2048 + 8), "BAD_ALIGN"),
    (dict(**{**Q8, "k_scales": (1 << 22) + 1}), "BAD_ALIGN")])
def test_pools_are_refused(change, code):
    """By every entry point that takes a pool, before any launch."""
    m, L = _lib()
    want = getattr(m, "KQ_ERR_" + code)
    p = ctypes.byref(_pool(**change))
    x = 1 << 26
    assert L.kq_paged_write(p, x, 1024, 128, x, 1024, 128, x, 4, None) == want
    assert L.kq_paged_read(p, x, 4, x, x, None) == want
    assert L.kq_sdpa_paged(p and x, 4096, p, x, 4, 4, x, x, 4, 2, 32, 4, 64, 0.1, x, 4096, None, 0, None) == want


def test_calls_are_refused():
    m, L = _lib()
    ok, x = ctypes.byref(_pool()), 1 << 26
    assert L.kq_paged_write(ok, None, 0, 0, None, 0, 0, None, 0, None) == m.KQ_OK  # nothing to write
    assert L.kq_paged_write(ok, None, 1024, 128, x, 1024, 128, x, 4, None) == m.KQ_ERR_NULL_POINTER
    assert L.kq_paged_write(ok, x, 1024, 128, x, 1024, 128, None, 4, None) == m.KQ_ERR_NULL_POINTER
    assert L.kq_paged_write(ok, x + 2, 1024, 128, x, 1024, 128, x, 4, None) == m.KQ_ERR_BAD_ALIGN
    assert L.kq_paged_write(ok, x, 1028, 128, x, 1024, 128, x, 4, None) == m.KQ_ERR_BAD_ALIGN
    assert L.kq_paged_write(ok, x, 1024, 128, x, 1024, 128, x, -1, None) == m.KQ_ERR_BAD_SHAPE
    assert L.kq_paged_write(ok, x, 1024, 128, x, 1024, 128, x, 1 << 25, None) == m.KQ_ERR_BAD_SHAPE
    assert L.kq_paged_read(ok, x, 4, None, x, None) == m.KQ_ERR_NULL_POINTER
    assert L.kq_paged_read(ok, x, 4, x + 8, x, None) == m.KQ_ERR_BAD_ALIGN

    def sdpa(**kw):
        d = dict(q=x, qs=4096, pool=ok, tab=x, ts=4, w=4, lens=x, cu=x, T=4, B=2, Hq=32, mq=4, mkv=64, out=x, os=4096,
                 ws=None, n=0)
        d.update(kw)
        return L.kq_sdpa_paged(d["q"], d["qs"], d["pool"], d["tab"], d["ts"], d["w"], d["lens"], d["cu"], d["T"], d["B"],
                               d["Hq"], d["mq"], d["mkv"], 0.1, d["out"], d["os"], d["ws"], d["n"], None)
    assert sdpa(T=0) == m.KQ_OK and sdpa(B=0) == m.KQ_OK
    for name in ("q", "tab", "lens", "cu", "out"):
        assert sdpa(**{name: None}) == m.KQ_ERR_NULL_POINTER, name
    for bad in (dict(T=-1), dict(B=-1), dict(Hq=12), dict(Hq=0), dict(Hq=8 * 65), dict(mq=0), dict(mkv=0), dict(w=0),
                dict(ts=3), dict(qs=4088), dict(os=4088), dict(T=1 << 26), dict(mkv=(1 << 30) + 1)):
        assert sdpa(**bad) == m.KQ_ERR_BAD_SHAPE, bad
    for bad in (dict(q=x + 8), dict(out=x + 2), dict(qs=4100), dict(os=4100)):
        assert sdpa(**bad) == m.KQ_ERR_BAD_ALIGN, bad
    need = L.kq_sdpa_paged_workspace_bytes(4, 2, 32, 8, 128, 4, 1 << 16, 0)
    assert need > 0
    assert sdpa(mkv=1 << 16) == m.KQ_ERR_WORKSPACE_TOO_SMALL
    assert sdpa(mkv=1 << 16, ws=x, n=need - 1) == m.KQ_ERR_WORKSPACE_TOO_SMALL
    assert sdpa(mkv=1 << 16, ws=x + 16, n=need) == m.KQ_ERR_BAD_ALIGN

    def plan(**kw):
        d = dict(seq=x, keep=None, new=x, B=2, tab=x, ts=4, w=4, st=x, n=8, cnt=x, ps=16, T=4, cu=x, kv=x, sl=x, pos=x,
                 left=x, ref=x)
        d.update(kw)
        return L.kq_paged_plan(d["seq"], d["keep"], d["new"], d["B"], d["tab"], d["ts"], d["w"], d["st"], d["n"], d["cnt"],
                               d["ps"], d["T"], d["cu"], d["kv"], d["sl"], d["pos"], d["left"], d["ref"], None)
    for name in ("seq", "new", "tab", "st", "cnt", "cu", "kv", "sl", "pos", "left", "ref"):
        assert plan(**{name: None}) == m.KQ_ERR_NULL_POINTER, name
    for bad in (dict(B=0), dict(B=2049), dict(w=0), dict(ts=3), dict(n=-1), dict(T=-1), dict(ps=8), dict(ps=24),
                dict(ps=2048), dict(w=1 << 28, ts=1 << 28), dict(B=2048, w=1 << 19, ts=1 << 19), dict(n=1 << 30)):
        assert plan(**bad) == m.KQ_ERR_BAD_SHAPE, bad


def test_workspace_follows_the_longest_rows():
    """One partial (D + 2 floats) a token, query head and split at most; none for
    rows of one split; bounded for prompt chunks however long."""
    _, L = _lib()

    def f(T, B, kv, mq):
        return L.kq_sdpa_paged_workspace_bytes(T, B, 32, 8, 128, mq, kv, 0)
    assert f(8, 8, 64, 1) == 0 and f(0, 8, 4096, 1) == 0
    assert 0 < f(8, 8, 4096, 1) <= f(8, 8, 131072, 1) <= 8 * 32 * 520 * 1024
    assert f(65536, 1, 131072, 65536) <= 128 << 20


def test_ops_refuse():
    from gmlx_amd import KQError, ops
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    sl = torch.zeros(3, dtype=torch.int32)
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    one = torch.zeros(1, dtype=torch.int32)
    tab = torch.zeros(1, 4, dtype=torch.int32)
    for call in (lambda: ops.paged_write(x, x, k, k, sl), lambda: ops.paged_read(k, k, sl),
                 lambda: ops.sdpa_paged(x, k, k, tab, one, torch.zeros(2, dtype=torch.int32), 0.1),
                 lambda: ops.paged_plan(one, one, tab, sl, one, 16, 4)):
        with pytest.raises(ValueError, match="GPU only"):
            call()


@pytest.mark.parametrize("name", ["paged_plan", "paged_write", "paged_read", "sdpa_paged"])
def test_faults_can_be_injected(name, monkeypatch):
    from gmlx_amd import KQError, ops
    monkeypatch.setenv("GMLX_HIP_FAULT", name)
    t = torch.zeros(1)
    args = {"paged_plan": (t, t, t, t, t, 16, 1), "paged_write": (t, t, t, t, t), "paged_read": (t, t, t),
            "sdpa_paged": (t, t, t, t, t, t, 1.0)}[name]
    with pytest.raises(KQError, match="fault injected"):
        getattr(ops, name)(*args)


def test_plan_reference_keeps_every_page_once():
    """Over many steps every page is in one row's table or on the stack."""
    rng = np.random.default_rng(0)
    B, page, n_pages, width = 6, 16, 40, 30
    seq, table = [0] * B, np.zeros((B, width), np.int32)
    stack, count = list(range(n_pages)), n_pages
    refusals = 0
    for _ in range(300):
        new = [int(x) for x in rng.integers(0, 60, B) * (rng.random(B) < 0.5)]
        keep = [0 if rng.random() < 0.15 else int(s - rng.integers(0, 5) * (s > 5)) for s in seq]
        cu, kv, slots, pos, count, refused, table, stack = ref.plan(seq, new, table, stack, count, page, sum(new), keep)
        refusals += sum(refused)
        seq = kv
        held = [int(p) for b in range(B) for p in table[b, :-(-seq[b] // page)]]
        assert sorted(held + list(stack[:count])) == list(range(n_pages))
        for b in range(B):
            if not refused[b]:
                for s, p in zip(slots[cu[b]:cu[b + 1]], pos[cu[b]:cu[b + 1]]):
                    assert s == table[b, p // page] * page + p % page
    assert refusals > 20


def _before_exec(text):
    """(kernel, label, instruction) of vector instructions between the start of a
    block that lanes join again and its restore of EXEC: those lanes would skip
    them.  Such blocks are where a `s_cbranch_execz` goes, and behind loops that
    lanes leave one by one."""
    joins = set(re.findall(r"s_cbranch_execz\s+(\.LBB\w+)", text))
    kernel = block = last = None
    found, seen = [], []
    for line in text.splitlines():
        name = re.match(r"([A-Za-z_]\w*):", line)
        label = re.match(r"(\.LBB\w+):|; (%bb\.\w+):", line)
        code = line.split(";")[0].strip()
        if name:
            kernel, block = name.group(1), None
        elif label:
            joined = label.group(1) in joins or (label.group(2) and last == "s_cbranch_execnz")
            block, seen = (label.group(0) if joined else None), []
        elif code and not code.startswith("."):
            last = code.split()[0]
            if block is None:
                continue
            if re.match(r"s_(or|andn2)_b64 exec, exec|s_mov_b64 exec|s_(or|andn2)_saveexec", code):
                found += [(kernel, block, x) for x in seen]
                block = None
            elif re.match(r"s_c?branch|s_and_saveexec|s_endpgm|s_barrier", code):
                block = None
            elif re.match(r"(v|ds|global|flat|buffer|scratch)_", code) and not re.match(r"v_(readlane|writelane|readfirstlane)", code):
                seen.append(code)
    return found


def test_register_copies_stand_behind_the_restore_of_exec(tmp_path):
    """Of the attention kernels as compiled: where the compiler splits a live
    range at a block that lanes join again, it can put the copy before the
    restore of EXEC, which lost addresses where no lane had been in the branch."""
    bad = "k:\n\ts_cbranch_execz .LBB0_2\n; %bb.1:\n\tv_mov_b32 v0, v1\n.LBB0_2:\n\tv_accvgpr_write_b32 a0, v2\n" \
          "\ts_or_b64 exec, exec, s[0:1]\n"
    assert _before_exec(bad) == [("k", ".LBB0_2:", "v_accvgpr_write_b32 a0, v2")]
    assert not _before_exec(bad.replace("\tv_accvgpr_write_b32 a0, v2\n", ""))
    from gmlx_amd import build
    out = tmp_path / "kq_paged.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "-S", os.path.join(build.CSRC, "kq_paged.hip"), "-o", str(out),
                    "--offload-device-only"], check=True, capture_output=True)
    text = out.read_text()
    assert "kq_paged_wave_kernel" in text
    assert not _before_exec(text)


def _sdpa(T, B, Hq, mkv, mq=None, ws=None, n=0, scale=0.1, **pool):
    """kq_sdpa_paged of a pool of pages, on addresses that no launch would get to."""
    m, L = _lib()
    x = 1 << 26
    return L.kq_sdpa_paged(x, Hq * 128, ctypes.byref(_pool(**pool)), x, 1 << 17, 1 << 17, x, x, T, B, Hq, mq or T, mkv, scale,
                           x, Hq * 128, ws, n, None)


@pytest.mark.parametrize("T,B,Hq", [(16384, 1, 64), (16384, 64, 64), (32768, 1, 32), (8192, 2048, 128), (1 << 20, 16, 8),
                                    (2048, 2048, 32)])
def test_long_prompts_over_long_tables_are_taken(T, B, Hq):
    """A chunk has few splits however many keys there may be: not refused, and
    its partials bounded (a million keys; asked without the workspace)."""
    m, L = _lib()
    need = L.kq_sdpa_paged_workspace_bytes(T, B, Hq, 8, 128, T, 1 << 20, 0)
    few = min(T, B * (16 // (Hq // 8)))  # tokens of rows of up to 16 columns, in splits of 512 keys
    assert 0 < need <= (few * Hq * 2048 + B * 512 * 128) * (128 * 4 + 8) + 256
    assert _sdpa(T, B, Hq, 1 << 20) == m.KQ_ERR_WORKSPACE_TOO_SMALL
    assert _sdpa(T, B, Hq, 1 << 20, ws=1 << 30, n=need - 1) == m.KQ_ERR_WORKSPACE_TOO_SMALL


def test_calls_past_31_bit_numbers_are_refused():
    """Partials, or waves, that 32-bit numbers cannot count."""
    m, L = _lib()
    for T, B, Hq, mq, kv in ((1 << 20, 1 << 20, 8, 1, 1 << 30), (1 << 19, 1 << 19, 8, 1, 1 << 27)):
        assert _sdpa(T, B, Hq, kv, mq=mq) == m.KQ_ERR_BAD_SHAPE
        assert L.kq_sdpa_paged_workspace_bytes(T, B, Hq, 8, 128, mq, kv, 0) == 0
    # arguments that the call refuses by themselves need no workspace either
    assert L.kq_sdpa_paged_workspace_bytes(2 ** 31 - 1, 4, 2 ** 31 - 1, 1, 128, 4, 2 ** 31 - 1, 0) == 0
    assert L.kq_sdpa_paged_workspace_bytes(4, 4, 8, 8, 128, 4, (1 << 30) + 1, 0) == 0


def test_workspace_counts_each_token_once():
    """A step of 300 rows, a prompt among them: tokens of rows of few columns at
    their splits, the rest at a chunk's (64 at most on 8 kv heads)."""
    _, L = _lib()
    T, B, Hq, few, many = 2348, 300, 32, 131072 // 512, 64
    need = L.kq_sdpa_paged_workspace_bytes(T, B, Hq, 8, 128, 2048, 131072, 0)
    assert 0 < need <= (4 * B * few + (T - 4 * B) * many) * Hq * (128 * 4 + 8) + 256


def test_writes_to_places_that_share_memory_are_refused():
    """Pools that repeat a page or a head (expanded views), or whose K is their V;
    they can be read and attended."""
    m, L = _lib()
    x = 1 << 26

    def write(**kw):
        return L.kq_paged_write(ctypes.byref(_pool(**kw)), x, 1024, 128, x, 1024, 128, x, 4, None)
    for kw in (dict(page_stride=0), dict(head_stride=0), dict(head_stride=128), dict(page_stride=16 * 128), dict(v=1 << 20),
               dict(**{**Q8, "v_scales": Q8["k_scales"]})):
        assert write(**kw) == m.KQ_ERR_BAD_ARGUMENT, kw
    # one page, one head: their strides are never used
    assert write(page_stride=0, n_pages=1, k=None) == m.KQ_ERR_NULL_POINTER
    for kw in (dict(head_stride=0), dict(page_stride=0), dict(v=1 << 20)):
        assert L.kq_paged_read(ctypes.byref(_pool(**kw)), x, 4, x + 8, x, None) == m.KQ_ERR_BAD_ALIGN


def test_scales_that_are_no_numbers_are_refused():
    """NaN, infinities, and what passes fp32 in the kernels' log2 units."""
    m, _ = _lib()
    for scale in (float("nan"), float("inf"), float("-inf"), 3e38, -3e38):
        assert _sdpa(4, 2, 32, 64, scale=scale) == m.KQ_ERR_BAD_ARGUMENT, scale


def test_once_for_each_device(tmp_path):
    """What launches need once is done on every device, and again after a failure."""
    from gmlx_amd import build
    (tmp_path / "t.cpp").write_text('''
#include "kq_once.h"
int main() {
    OncePerDevice once;
    int calls = 0;
    const auto ok = [&] { return ++calls > 0; };
    if (!once(0, ok) || !once(0, ok) || calls != 1) return 1;
    if (!once(1, ok) || calls != 2 || !once(63, ok) || calls != 3) return 2;
    if (once(2, [&] { ++calls; return false; }) || calls != 4) return 3;
    if (!once(2, ok) || !once(2, ok) || calls != 5) return 4;
    if (!once(64, ok) || !once(64, ok) || calls != 7) return 5;  // (past the table: at every call)
    if (once(-1, ok) || calls != 7) return 6;
    return 0;
}
''')
    subprocess.run(["g++", "-std=c++17", "-I", build.CSRC, str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    assert subprocess.run([str(tmp_path / "t")]).returncode == 0


def test_8bit_pools_of_tokens_before_heads_are_refused_by_name():
    """Their scales lie a 64th of the way, but a head's tokens do not lie one after
    the other; with one kv head they do."""
    from gmlx_amd import ops

    def layout(H):
        k = torch.zeros(4, 16, H, 128, dtype=torch.uint8).permute(0, 2, 1, 3)
        s = torch.zeros(4, 16, H, 2, dtype=torch.float16).permute(0, 2, 1, 3)
        return ops._PoolLayout(k, k, (s, s, s, s))
    with pytest.raises(ValueError, match="8-bit pool's tokens"):
        layout(2)
    assert layout(1).q8 == 1


def test_register_copies_of_the_decode_kernels(tmp_path):
    """The same of the kernels over contiguous caches."""
    from gmlx_amd import build
    out = tmp_path / "kq_attention.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "-S", os.path.join(build.CSRC, "kq_attention.hip"), "-o", str(out),
                    "--offload-device-only"], check=True, capture_output=True)
    text = out.read_text()
    assert "kq_sdpa_split_kernel" in text
    assert not _before_exec(text)


def test_plan_refuses_more_tokens_than_its_grid_counts():
    """A grid's step past 2^31 - 1 tokens would be a negative number."""
    m, L = _lib()
    x = 1 << 26
    for tokens in ((1 << 30) + 1, (1 << 31) - 1):
        assert L.kq_paged_plan(x, None, x, 2, x, 4, 4, x, 8, x, 16, tokens, x, x, x, x, x, x, None) == m.KQ_ERR_BAD_SHAPE
