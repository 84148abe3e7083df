"""The anchor layers' host side, with no GPU: include/kdn_anchor.h and its mirrors, argument errors, the pages' bookkeeping,
and the oracle's gradients against differences."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from kdn import _native as N
from kdn import anchor
from oracle import anchor as oa

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "kdn_anchor.h")
P = 16


def test_header_declares_what_the_library_exports():
    text = open(HEADER).read()
    declared = sorted(set(re.findall(r"^\s*(?:int|int64_t|size_t|void)\s+(kdn_\w+)\s*\(", text, re.M)))
    assert declared == sorted(N.ANCHOR_EXPORTED)
    out = subprocess.run(["nm", "-D", "--defined-only", N.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert set(declared) <= set(re.findall(r"\sT\s+(kdn_\w+)$", out, re.M))
    assert N.lib().kdn_anchor_version() == 1 << 16


@pytest.mark.parametrize("cname,mirror", [("kdn_attn_args", N.AttnArgs), ("kdn_attn_bwd_args", N.AttnBwdArgs), ("kdn_rotary_args", N.RotaryArgs),
                                          ("kdn_page_append_args", N.PageAppendArgs), ("kdn_tree_attn_args", N.TreeAttnArgs)])
def test_struct_layouts(cname, mirror, tmp_path):
    fields = [f[0] for f in mirror._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'printf("%zu\\n", sizeof({cname}));',
           *(f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields), "return 0;}"]
    (tmp_path / "l.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-std=c99", "-o", tmp_path / "l", tmp_path / "l.c"], check=True)
    got = [int(x) for x in subprocess.run([tmp_path / "l"], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror), *(getattr(mirror, f).offset for f in fields)]


@pytest.mark.parametrize("packed,mirror", [(anchor._ATTN, N.AttnArgs), (anchor._ATTN_BWD, N.AttnBwdArgs), (anchor._ROTARY, N.RotaryArgs),
                                           (anchor._APPEND, N.PageAppendArgs), (anchor._TREE, N.TreeAttnArgs)])
def test_packed_arguments_are_the_mirrors(packed, mirror):
    """Numbers 1, 2, ... packed in order read back from the mirror's fields in order (arrays flattened)."""
    n = len(packed.unpack(bytes(packed.size)))
    a = mirror.from_buffer_copy(packed.pack(*range(1, n + 1)).ljust(ctypes.sizeof(mirror), b"\0"))
    got = []
    for name, _ in mirror._fields_:
        x = getattr(a, name)
        got += list(x) if isinstance(x, ctypes.Array) else [x]
    assert got == list(range(1, n + 1))


def _attn(**kw):
    a = N.AttnArgs()
    a.num_seqs, a.total_q, a.total_k, a.H, a.H_kv, a.d, a.dtype, a.scale = 1, 8, 8, 4, 2, 64, 1, 0.125
    a.cu_q = a.q = a.k = a.v = a.y = 1 << 12  # never read: every case below is refused
    for s in ("q", "k", "v", "y"):
        getattr(a, s + "_stride")[0], getattr(a, s + "_stride")[1] = 256, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status", [(dict(H=5), -1), (dict(H_kv=0), -1), (dict(dtype=7), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1),
                                       (dict(scale=float("inf")), -1), (dict(num_seqs=-1), -1), (dict(d=96), -2), (dict(total_k=9), -1),
                                       (dict(q=None), -1), (dict(y=None), -1), (dict(cu_q=None), -1), (dict(v=(1 << 12) + 2), -4),
                                       (dict(q_stride=N._i64x2(257, 64)), -4), (dict(total_q=1 << 40, total_k=1 << 40), -2)])
def test_attention_arguments(kw, status):
    a = _attn(**kw)
    assert N.lib().kdn_attn_fwd(ctypes.byref(a), None) == status
    if status != -4:
        b = N.AttnBwdArgs()
        b.fwd = ctypes.addressof(a)
        b.dy = b.dq = b.dk = b.dv = b.workspace = 1 << 12
        a.lse, b.workspace_bytes = 1 << 12, 1 << 20
        assert N.lib().kdn_attn_bwd(ctypes.byref(b), None) == status


def test_backward_arguments():
    a = _attn(lse=1 << 12)
    b = N.AttnBwdArgs()
    b.fwd = ctypes.addressof(a)
    assert N.lib().kdn_attn_bwd_workspace_bytes(ctypes.byref(b)) == 1024 + 2 * 2 * 8 * 2 * 64 * 4  # lse and delta; dk and dv of two heads each
    assert N.lib().kdn_attn_bwd(ctypes.byref(b), None) == -1  # no dy
    b.dy = b.dq = b.dk = b.dv = b.workspace = 1 << 12
    b.workspace_bytes = 1024 + 2 * 2 * 8 * 2 * 64 * 4 - 1
    assert N.lib().kdn_attn_bwd(ctypes.byref(b), None) == -3
    assert N.lib().kdn_attn_bwd(None, None) == -1
    b.fwd = None
    assert N.lib().kdn_attn_bwd(ctypes.byref(b), None) == -1 and N.lib().kdn_attn_bwd_workspace_bytes(ctypes.byref(b)) == 0


def test_rotary_arguments():
    def call(**kw):
        a = N.RotaryArgs()
        a.tokens, a.H, a.H_kv, a.d, a.rotary_dim, a.dtype, a.magnitude = 2, 4, 2, 64, 64, 1, 1.0
        a.positions = a.inv_freq = a.q = a.k = a.q_out = a.k_out = 1 << 12
        for k, v in kw.items():
            setattr(a, k, v)
        return N.lib().kdn_rotary(ctypes.byref(a), None)

    assert [call(rotary_dim=r) for r in (0, 63, 66)] == [-1] * 3
    assert [call(d=32, rotary_dim=32), call(positions=None), call(k=None), call(magnitude=float("nan")), call(q=8)] == [-2, -1, -1, -1, -4]
    assert call(tokens=0) == 0


def test_page_arguments():
    L = N.lib()
    pairs = (ctypes.c_int32 * 4)(0, 1, 1, 2)
    assert L.kdn_page_copy(4096, 4, 64, pairs, 2, None) == -1        # a target that is a source
    assert L.kdn_page_copy(4096, 4, 60, pairs, 1, None) == -1
    assert L.kdn_page_copy(4100, 4, 64, pairs, 1, None) == -4
    assert L.kdn_page_copy(None, 4, 64, pairs, 1, None) == -1
    assert L.kdn_page_copy(4096, 4, 64, pairs, 9, None) == -1        # more targets than pages
    assert L.kdn_page_copy(None, 4, 64, None, 0, None) == 0
    h = ctypes.c_void_p()
    for pages, tokens, streams in ((0, 16, 1), (4, 8, 1), (4, 24, 1), (4, 16, 0)):
        assert L.kdn_page_pool_create(pages, tokens, streams, ctypes.byref(h)) == -1 and not h.value
    a = N.PageAppendArgs()
    a.tokens, a.H_kv, a.d, a.dtype, a.page_tokens, a.num_pages = 1, 1, 64, 1, 24, 4
    assert L.kdn_page_append(ctypes.byref(a), None) == -2
    a.page_tokens = 16
    assert L.kdn_page_append(ctypes.byref(a), None) == -1


def test_tree_arguments():
    def args(**kw):
        a = N.TreeAttnArgs()
        a.num_seqs, a.total_new, a.max_new, a.max_context, a.H, a.H_kv, a.d, a.dtype, a.scale = 2, 2, 1, 4096, 8, 2, 128, 1, 0.1
        a.page_tokens, a.num_pages, a.table_width, a.table_stride = 16, 999, 256, 256
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    size, call = N.lib().kdn_tree_attn_workspace_bytes, N.lib().kdn_tree_attn
    for bad in (dict(max_new=65), dict(page_tokens=8), dict(page_tokens=48), dict(d=96)):
        assert size(args(**bad)) == 0 and call(args(**bad), None) == -2
    for bad in (dict(max_new=0), dict(max_context=4097), dict(num_pages=0), dict(H=9), dict(scale=-1.0)):
        assert size(args(**bad)) == 0 and call(args(**bad), None) == -1
    assert call(args(), None) == -1  # no tensors
    assert call(args(num_seqs=0), None) == 0
    grows = [size(args(num_seqs=n, max_context=c)) for n in (1, 2, 7, 8, 9, 64, 300) for c in (4096,)]
    assert grows == sorted(grows)
    grows = [size(args(max_context=c)) for c in (0, 1, 128, 129, 1000, 4096)]
    assert grows == sorted(grows) and grows[0] == 16


def test_forks_share_pages_until_one_writes():
    pool = anchor.PagePool(8, P, 4)
    a = pool.open()
    assert pool.extend(a, 40) == [] and pool.table([a]).tolist() == [[0, 1, 2]] and pool.used == 3
    b = pool.fork(a)
    assert pool.used == 3 and pool.length(b) == 40
    assert pool.extend(b, 1) == [(2, 3)] and pool.table([a, b]).tolist() == [[0, 1, 2], [0, 1, 3]]
    assert pool.extend(a, 9) == [] and pool.table([a]).tolist() == [[0, 1, 2, 4]]  # page 2 is a's alone now
    c = pool.fork(a)
    pool.truncate(c, 32)
    assert pool.extend(c, 1) == [] and pool.table([c]).tolist() == [[0, 1, 5]]      # full pages are shared, not copied
    pool.truncate(c, 20)
    assert pool.extend(c, 1) == [(1, 5)]                                            # a shared page, partly kept
    assert pool.rows(b, 38, 3).tolist() == [3 * P + 6, 3 * P + 7, 3 * P + 8]
    pool.close(a)
    assert pool.used == 4
    pool.close(b)
    pool.close(c)
    assert pool.used == 0 and pool.free == 8


def test_pool_capacity_errors_change_nothing():
    pool = anchor.PagePool(3, P, 2)
    a = pool.open()
    pool.extend(a, 20)
    b = pool.fork(a)
    with pytest.raises(RuntimeError):
        pool.open()
    with pytest.raises(RuntimeError):
        pool.fork(a)
    with pytest.raises(RuntimeError):
        pool.extend(b, 20)      # its own last page and one more: one is free
    assert pool.length(b) == 20 and pool.free == 1 and pool.table([a]).tolist() == pool.table([b]).tolist()
    assert pool.extend(b, 1) == [(1, 2)]
    for call in (lambda: pool.extend(b, -1), lambda: pool.truncate(b, 22), lambda: pool.rows(b, 20, 2), lambda: pool.close(7),
                 lambda: pool.extend(9, 1), lambda: pool.length(-1)):
        with pytest.raises(RuntimeError):
            call()
    pool.close(b)
    with pytest.raises(RuntimeError):
        pool.close(b)
    assert pool.open() == b and pool.length(b) == 0 and pool.table([b]).shape == (1, 0)


def test_compaction():
    pool = anchor.PagePool(10, P, 4)
    s = [pool.open() for _ in range(3)]
    for x in s:
        pool.extend(x, 3 * P)
    t = pool.fork(s[2])
    pool.close(s[0])
    pool.truncate(s[1], P)
    moves = pool.compact()
    assert pool.used == 4 and sorted(moves[:, 0].tolist()) == [6, 7, 8] and sorted(moves[:, 1].tolist()) == [0, 1, 2]
    assert pool.table([s[2]]).tolist() == pool.table([t]).tolist()
    assert {int(x) for x in pool.table([s[1], s[2]]).flatten()} <= set(range(4))
    assert pool.compact().shape == (0, 2)
    few = (ctypes.c_int32 * 2)()
    pool.extend(s[1], 3 * P)
    pool.close(s[2])
    pool.close(t)
    before = pool.table([s[1]]).tolist()
    assert N.lib().kdn_page_pool_compact(pool._h, few, 1) == N.KDN_ERR_CAPACITY  # no room for the list: nothing moved
    assert pool.table([s[1]]).tolist() == before == [[3, 4, 5, 6]]
    assert pool.compact().shape[0] == 3 and sorted(pool.table([s[1]])[0].tolist()) == [0, 1, 2, 3]


def test_frequencies():
    f, m = anchor.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f[0] == 1 and abs(float(f[-1]) - 10000.0 ** (-62 / 64)) < 1e-18 and m == 1
    assert torch.allclose(anchor.rotary_frequencies(64, scaling="linear", factor=4)[0], f / 4, rtol=1e-15)
    b = anchor.rotary_frequencies(64, scaling="base", factor=4)[0]
    assert abs(float(b[-1] / f[-1]) - 0.25) < 1e-12 and b[0] == 1
    p, m = anchor.rotary_frequencies(64, scaling="parts", factor=4, trained_length=4096)
    assert p[0] == f[0] and abs(float(p[-1] / f[-1]) - 0.25) < 1e-12 and (p <= f).all() and (p >= f / 4).all() and m > 1


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    cu, ck = [0, 3, 3, 8], [0, 5, 6, 8]
    x = [torch.randn(n, h, 4, generator=g, dtype=torch.float64) for n, h in ((8, 4), (8, 2), (8, 2))]
    dy = torch.randn(8, 4, 4, generator=g, dtype=torch.float64)
    r = oa.attention(*x, cu, ck, dy=dy)
    h = 1e-6
    for i, name in enumerate(("dq", "dk", "dv")):
        u = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        f = [float((oa.attention(*(t + s * u if j == i else t for j, t in enumerate(x)), cu, ck)["y"] * dy).sum()) for s in (h, -h)]
        want = float((r[name] * u).sum())
        assert abs((f[0] - f[1]) / (2 * h) - want) < 1e-7 * (1 + abs(want))


def test_oracle_rows_that_see_nothing():
    r = oa.attention(torch.ones(4, 1, 4), torch.ones(1, 1, 4), torch.ones(1, 1, 4), [0, 4], [0, 1], dy=torch.ones(4, 1, 4))
    assert not r["y"][:3].any() and r["y"][3].eq(1).all() and torch.isneginf(r["lse"][0, :3]).all() and not r["dq"][:3].any()


def test_hybrid_pool_bookkeeping_on_the_host():
    from serving import HybridMemoryPool
    pool = HybridMemoryPool(4, 64, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device="cpu", anchor_layers=2, anchor_heads=1,
                            anchor_pages=6)
    a = pool.allocate_stream(20)
    plan = pool.anchor_plan([a], [20])
    assert plan.rows.tolist() == list(range(20)) and plan.positions.tolist() == list(range(20)) and plan.context_lens.tolist() == [0]
    b = pool.fork_stream(a)
    plan = pool.anchor_plan([b, a], [1, 2])
    assert plan.rows.tolist() == [2 * P + 4, P + 4, P + 5] and plan.cu_seqlens.tolist() == [0, 1, 3] and plan.context_lens.tolist() == [20, 20]
    assert plan.page_table.tolist() == [[0, 2], [0, 1]] and (plan.max_new, plan.max_context) == (2, 20)
    plan = pool.anchor_plan([a, b], [2, 1], depths=[0, 1, 0])
    assert plan.positions.tolist() == [22, 23, 21] and plan.rows is None and pool.anchor_tokens(a) == 22
    with pytest.raises(RuntimeError):
        pool.anchor_plan([a, b], [30, 40])  # five pages where three are free
    assert (pool.anchor_tokens(a), pool.anchor_tokens(b), pool.anchor_pages_free) == (22, 21, 3)
    with pytest.raises(ValueError):
        pool.anchor_plan([a, a], [1, 1])
    pool.release_stream(a)
    assert pool.anchor_pages_used == 2 and pool.anchor_compact() == 1  # pages 0 and 2 are b's
    assert pool.anchor_plan([b], [1]).page_table.tolist() == [[0, 1]]
    assert HybridMemoryPool(2, 64, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device="cpu").anchor_layers == 0


@pytest.mark.timeout(900)
def test_host_paths_clean_under_asan_and_ubsan(tmp_path):
    """The argument checks and the pages' bookkeeping above, in a child process, against the library with its host code
    instrumented (as tests/test_host_sanitizers.py does for the rest)."""
    import sys
    from kdn import build as kbuild
    runtime = kbuild.asan_runtime()
    if os.environ.get("KDN_LIBRARY") or not runtime or not os.path.exists(kbuild.hipcc()):
        pytest.skip("hipcc's ASan runtime is not installed, or this is the child")
    lib = kbuild.build_host_sanitized(str(tmp_path / "hostsan"))
    env = dict(os.environ, KDN_LIBRARY=lib, LD_PRELOAD=runtime, UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1:exitcode=87",
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:abort_on_error=0:exitcode=86")
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-m", "not gpu", "-p", "no:cacheprovider", __file__], cwd=REPO, env=env,
                         capture_output=True, text=True, timeout=600)
    report = res.stdout[-3000:] + res.stderr[-3000:]
    assert res.returncode == 0 and "ERROR: AddressSanitizer" not in report and "runtime error" not in report, report
    assert " passed" in report or res.stdout.count(".") >= 30, report
