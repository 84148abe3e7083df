"""The host side of the bounded contexts, with no GPU: include/kdn_bounded.h and its mirrors, argument errors, the pages'
bookkeeping for windows and eviction, and the oracle against the plainest forms."""
import ctypes
import os
import random
import re
import subprocess

import pytest
import torch

from kdn import _native as N
from kdn import anchor, bounded
from layers import AnchorAttentionLayer
from oracle import anchor as oa
from oracle import bounded as ob
from serving import HybridMemoryPool

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "kdn_bounded.h")


def test_header_declares_what_the_library_exports():
    text = open(HEADER).read()
    declared = sorted(set(re.findall(r"^\s*(?:int|int64_t|size_t|void)\s+(kdn_\w+)\s*\(", text, re.M)))
    assert declared == sorted(N.BOUNDED_EXPORTED)
    out = subprocess.run(["nm", "-D", "--defined-only", N.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert set(declared) <= set(re.findall(r"\sT\s+(kdn_\w+)$", out, re.M))
    assert N.lib().kdn_bounded_version() == 1 << 16


@pytest.mark.parametrize("cname,mirror,packed", [("kdn_tree_bound_args", N.TreeBoundArgs, anchor._BOUND),
                                                 ("kdn_attn_weights_args", N.AttnWeightsArgs, bounded._WEIGHTS),
                                                 ("kdn_evict_args", N.EvictArgs, bounded._EVICT)])
def test_struct_layouts(cname, mirror, packed, tmp_path):
    fields = [f[0] for f in mirror._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'printf("%zu\\n", sizeof({cname}));',
           *(f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields), "return 0;}"]
    (tmp_path / "l.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-std=c99", "-o", tmp_path / "l", tmp_path / "l.c"], check=True)
    got = [int(x) for x in subprocess.run([tmp_path / "l"], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror), *(getattr(mirror, f).offset for f in fields)]
    n = len(packed.unpack(bytes(packed.size)))
    a = mirror.from_buffer_copy(packed.pack(*range(1, n + 1)).ljust(ctypes.sizeof(mirror), b"\0"))
    back = []
    for name, _ in mirror._fields_:
        x = getattr(a, name)
        back += list(x) if isinstance(x, ctypes.Array) else [x]
    assert back == list(range(1, n + 1))


def _attn(**kw):
    a = N.AttnArgs()
    a.num_seqs, a.total_q, a.total_k, a.H, a.H_kv, a.d, a.dtype, a.scale = 1, 8, 8, 4, 2, 64, 1, 0.125
    a.cu_q = a.q = a.k = a.v = a.y = 1 << 12  # never read: every case below is refused
    for s in ("q", "k", "v", "y"):
        getattr(a, s + "_stride")[0], getattr(a, s + "_stride")[1] = 256, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_window_arguments():
    L, a = N.lib(), _attn()
    b = N.AttnBwdArgs()
    b.fwd = ctypes.addressof(a)
    for window, sinks in ((0, 0), (-1, 0), (4, -1)):
        assert L.kdn_attn_window_fwd(ctypes.byref(a), window, sinks, None) == -1
        assert L.kdn_attn_window_bwd(ctypes.byref(b), window, sinks, None) == -1
        assert L.kdn_attn_window_bwd_workspace_bytes(ctypes.byref(b), window, sinks) == 0
    assert L.kdn_attn_window_fwd(ctypes.byref(_attn(d=96)), 4, 0, None) == -2
    assert L.kdn_attn_window_fwd(ctypes.byref(_attn(q=None)), 4, 0, None) == -1
    assert L.kdn_attn_window_bwd(None, 4, 0, None) == -1 and L.kdn_attn_window_fwd(None, 4, 0, None) == -1
    size = lambda w, s: L.kdn_attn_window_bwd_workspace_bytes(ctypes.byref(b), w, s)  # noqa: E731
    none = L.kdn_attn_bwd_workspace_bytes(ctypes.byref(b))
    assert size(8, 0) == size(4, 4) == size(2 ** 62, 2 ** 62) == size(4, 0) == none  # no window, or none with sinks
    assert size(4, 3) == none + 2 * (8 // 1024 + 3 + 1) * 2 * 3 * 2 * 64 * 4         # slots and sequences, subsets, sinks, heads
    long = _attn(total_q=4096, total_k=4096)
    g = N.AttnBwdArgs()
    g.fwd = ctypes.addressof(long)
    assert L.kdn_attn_window_bwd_workspace_bytes(ctypes.byref(g), 64, 257) == L.kdn_attn_bwd_workspace_bytes(ctypes.byref(g))  # no segments
    b.workspace, b.workspace_bytes, a.lse = 1 << 12, size(4, 3) - 1, 1 << 12
    b.dy = b.dq = b.dk = b.dv = 1 << 12
    assert L.kdn_attn_window_bwd(ctypes.byref(b), 4, 3, None) == -3


def _tree(**kw):
    a = N.TreeAttnArgs()
    a.num_seqs, a.total_new, a.max_new, a.max_context, a.H, a.H_kv, a.d, a.dtype, a.scale = 2, 2, 1, 4096, 8, 2, 128, 1, 0.1
    a.page_tokens, a.num_pages, a.table_width, a.table_stride = 16, 999, 256, 256
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bound(**kw):
    b = N.TreeBoundArgs()
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def test_tree_bound_arguments():
    size, call = N.lib().kdn_tree_attn_bounded_workspace_bytes, N.lib().kdn_tree_attn_bounded
    some = dict(weights=1 << 12, places=4100, num_slots=2)
    for a, b, status in ((_tree(), _bound(window=-1), -1), (_tree(), _bound(sinks=-1), -1), (_tree(d=96), _bound(window=4), -2),
                         (_tree(parents=1 << 12), _bound(**some), -1), (_tree(max_new=9), _bound(**some), -2),
                         (_tree(), _bound(**{**some, "places": -1}), -1), (_tree(), _bound(**{**some, "num_slots": 1}), -1),
                         (_tree(), _bound(**{**some, "weights": 4097}), -4), (_tree(), _bound(**{**some, "num_slots": 1 << 40}), -2)):
        assert size(ctypes.byref(a), ctypes.byref(b)) == 0 and call(ctypes.byref(a), ctypes.byref(b), None) == status
    assert call(ctypes.byref(_tree()), None, None) == -1 and size(None, ctypes.byref(_bound())) == 0
    plain = N.lib().kdn_tree_attn_workspace_bytes(ctypes.byref(_tree()))
    assert size(ctypes.byref(_tree()), ctypes.byref(_bound())) == plain == size(ctypes.byref(_tree()), ctypes.byref(_bound(window=4097)))
    assert size(ctypes.byref(_tree()), ctypes.byref(_bound(window=64))) == 16  # one chunk
    assert size(ctypes.byref(_tree()), ctypes.byref(_bound(**some))) == plain + 2 * 2 * 4 * (4096 + 32 + 128 + 2) * 4 + 32
    huge = _tree(num_seqs=1 << 20, H=1 << 12, H_kv=1 << 10)
    assert size(ctypes.byref(huge), ctypes.byref(_bound(**{**some, "num_slots": 1 << 20}))) == 0


def test_weights_arguments():
    def args(**kw):
        a = N.AttnWeightsArgs()
        a.num_seqs, a.total_q, a.total_k, a.H, a.H_kv, a.d, a.dtype, a.scale = 1, 8, 8, 4, 2, 64, 1, 0.125
        a.cu_q = a.q = a.k = a.lse = a.weights = 1 << 12
        a.places, a.num_slots = 8, 1
        for s in ("q", "k"):
            getattr(a, s + "_stride")[0], getattr(a, s + "_stride")[1] = 256, 64
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    size, call = N.lib().kdn_attn_weights_workspace_bytes, N.lib().kdn_attn_weights
    for kw, status in ((dict(H=5), -1), (dict(dtype=9), -1), (dict(scale=float("nan")), -1), (dict(window=-1), -1), (dict(sinks=-1), -1),
                       (dict(d=32), -2), (dict(total_k=9), -1), (dict(num_slots=0), -1), (dict(places=-1), -1), (dict(total_q=1 << 40, total_k=1 << 40), -2)):
        assert size(args(**kw)) == 0 and call(args(**kw), None) == status
    for kw, status in ((dict(q=None), -1), (dict(lse=None), -1), (dict(weights=None), -1), (dict(k=8), -4), (dict(q_stride=N._i64x2(257, 64)), -4)):
        assert size(args(**kw)) > 0 and call(args(**kw), None) == status
    assert size(args()) == 4  # few rows: no partial sums
    long = dict(total_q=4096, total_k=4096)
    assert 4 < size(args(**long)) <= 16 * 2 * 4096 * 4 and call(args(**long), None) == -3  # workgroups that share a tile, and no workspace
    sinks = size(args(window=64, sinks=9, **long)) - size(args(window=64, **long))  # partial sums of the rows far behind the sinks
    assert sinks > 0 and sinks % (2 * 9 * 4) == 0 and size(args(window=64, sinks=4032, **long)) == size(args(**long))
    for kw in (dict(window=64, sinks=9, num_seqs=1 << 30, num_slots=1 << 30, H=1 << 20, H_kv=1 << 20), dict(window=1, sinks=1 << 29, total_k=1 << 30, total_q=1 << 30),
               dict(window=1, sinks=1 << 29, total_k=1 << 30, total_q=1 << 30, num_seqs=1 << 30, num_slots=1 << 30, H=1 << 20, H_kv=1 << 20),
               dict(window=2 ** 62, sinks=2 ** 62)):
        assert size(args(**kw)) > 0
    assert call(args(num_seqs=0, num_slots=0), None) == 0 and call(args(total_k=0, total_q=0), None) == 0


def test_evict_arguments():
    def args(**kw):
        a = N.EvictArgs()
        a.num_seqs, a.layers, a.H_kv, a.d, a.dtype, a.page_tokens, a.num_pages, a.table_width, a.max_len = 2, 3, 4, 64, 1, 16, 99, 4, 64
        a.page_table = a.lens = a.keep = a.k_pages = a.v_pages = a.weights = a.positions = a.workspace = 1 << 12
        a.places, a.num_slots, a.workspace_bytes = 64, 2, 1 << 20
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    size, call = N.lib().kdn_evict_workspace_bytes, N.lib().kdn_evict
    for kw, status in ((dict(layers=0), -1), (dict(H_kv=0), -1), (dict(d=96), -2), (dict(page_tokens=24), -2), (dict(page_tokens=8), -2),
                       (dict(max_len=65), -1), (dict(places=63), -1), (dict(num_pages=0), -1), (dict(num_slots=1), -1), (dict(sinks=-1), -1),
                       (dict(recent=-1), -1), (dict(max_len=1 << 31, table_width=1 << 40, places=1 << 40), -2), (dict(num_seqs=1 << 29, num_slots=1 << 29), -2)):
        assert size(args(**kw)) == 0 and call(args(**kw), None) == status
    assert size(args()) == 24 * 4 * (1 + 2 * 32) + 16
    for kw, status in ((dict(lens=None), -1), (dict(positions=None), -1), (dict(workspace=None), -3), (dict(workspace_bytes=24 * 4 * 65 + 15), -3),
                       (dict(k_pages=8), -4), (dict(v_pages_stride=N._i64x4(0, 0, 0, 4)), -4)):
        assert call(args(**kw), None) == status
    assert call(args(num_seqs=0), None) == 0 and call(args(max_len=0), None) == 0


def test_grids_past_32_bits_of_work_items_are_refused():
    """Before anything is launched: such a grid would be cut short without an error."""
    L, none = N.lib(), ctypes.c_void_p(None)
    many = dict(num_seqs=1 << 20, H=32, H_kv=32)  # a tile slot a sequence and head: 33 million workgroups of 256
    for kw in (many, dict(many, dtype=0), dict(many, d=128)):
        assert L.kdn_attn_fwd(ctypes.byref(_attn(**kw)), none) == -2
        assert L.kdn_attn_window_fwd(ctypes.byref(_attn(**kw)), 4, 1, none) == -2
        fwd = _attn(lse=1 << 12, **kw)
        b = N.AttnBwdArgs()
        b.fwd = ctypes.addressof(fwd)
        b.dy = b.dq = b.dk = b.dv = b.workspace = 1 << 12
        b.workspace_bytes = 1 << 50
        for s in ("dy", "dq", "dk", "dv"):
            getattr(b, s + "_stride")[0], getattr(b, s + "_stride")[1] = 256, 64
        assert L.kdn_attn_bwd(ctypes.byref(b), none) == -2 and L.kdn_attn_window_bwd(ctypes.byref(b), 4, 1, none) == -2
    t = _tree(num_seqs=1 << 20, total_new=1 << 20, H=32, H_kv=32, max_context=128)
    t.cu_new = t.context_lens = t.page_table = t.q = t.k = t.v = t.y = t.k_pages = t.v_pages = t.workspace = 1 << 12
    for s in ("q", "k", "v", "y"):
        getattr(t, s + "_stride")[0], getattr(t, s + "_stride")[1] = 4096, 128
    t.workspace_bytes = 1 << 50
    for d, dtype in ((64, 1), (128, 1), (64, 0)):
        t.d, t.dtype, t.num_seqs = d, dtype, 1 << 21
        assert L.kdn_tree_attn(ctypes.byref(t), none) == -2 and L.kdn_tree_attn_bounded(ctypes.byref(t), ctypes.byref(_bound(window=4)), none) == -2
    t.max_new = 64  # more than 32 rows
    assert L.kdn_tree_attn(ctypes.byref(t), none) == -2
    w = N.AttnWeightsArgs()
    w.num_seqs, w.total_q, w.total_k, w.H, w.H_kv, w.d, w.dtype, w.scale = 1 << 20, 8, 8, 32, 32, 64, 0, 0.125
    w.cu_q = w.q = w.k = w.lse = w.weights = w.workspace = 1 << 12
    w.places, w.num_slots, w.workspace_bytes = 8, 1 << 20, 1 << 50
    assert L.kdn_attn_weights(ctypes.byref(w), none) == -2
    r = N.RotaryArgs()
    r.tokens, r.H, r.H_kv, r.d, r.rotary_dim, r.dtype, r.magnitude = 1 << 27, 4, 2, 64, 64, 1, 1.0
    r.positions = r.inv_freq = r.q = r.k = r.q_out = r.k_out = 1 << 12
    for s in ("q", "k", "q_out", "k_out"):
        getattr(r, s + "_stride")[0], getattr(r, s + "_stride")[1] = 256, 64
    assert L.kdn_rotary(ctypes.byref(r), none) == -2
    p = N.PageAppendArgs()
    p.tokens, p.H_kv, p.d, p.dtype, p.page_tokens, p.num_pages = 1 << 26, 8, 64, 1, 16, 4
    p.rows = p.k = p.v = p.k_pages = p.v_pages = 1 << 12
    assert L.kdn_page_append(ctypes.byref(p), none) == -2


def test_evict_refuses_rows_that_lie_on_one_another():
    a = N.EvictArgs()
    a.num_seqs, a.layers, a.H_kv, a.d, a.dtype, a.page_tokens, a.num_pages, a.table_width, a.max_len = 1, 2, 2, 64, 1, 16, 9, 4, 64
    a.page_table = a.lens = a.keep = a.k_pages = a.v_pages = a.weights = a.positions = a.workspace = 1 << 12
    a.places, a.num_slots, a.workspace_bytes = 64, 2, 1 << 20
    strides = dict(k_pages=(8192, 4096, 1024, 64), v_pages=(8192, 4096, 1024, 64), weights=(256, 128, 64), positions=(256, 128, 64))
    for name in strides:
        for i in range(len(strides[name])):
            for n, s in strides.items():
                for j, x in enumerate(s):
                    getattr(a, n + "_stride")[j] = 0 if (n, j) == (name, i) else x
            assert N.lib().kdn_evict(ctypes.byref(a), None) == -1


def test_pages_of_ones_own_and_dropped_ones():
    pool = anchor.PagePool(12, 16, 8)
    a = pool.open()
    pool.extend(a, 70)  # five pages
    assert pool.own(a, 70).shape == (0, 2) and pool.own(a, 0).shape == (0, 2)
    b = pool.fork(a)
    before = pool.table([a])[0].tolist()
    pairs = pool.own(b, 33)  # three pages
    assert pairs[:, 0].tolist() == before[:3] and pool.used == 8
    assert pool.table([b])[0].tolist() == pairs[:, 1].tolist() + before[3:] and pool.table([a])[0].tolist() == before
    assert pool.own(a, 33).shape == (0, 2)
    c = pool.fork(a)
    with pytest.raises(RuntimeError):
        pool.own(c, 70)  # five pages of four
    assert pool.used == 8 and pool.table([c])[0].tolist() == before
    with pytest.raises(RuntimeError):
        pool.own(c, 71)
    pool.close(c)
    pool.drop(b, 1, 3)
    assert pool.length(b) == 22 and pool.table([b])[0].tolist() == [int(pairs[0, 1]), before[4]] and pool.used == 6
    pool.drop(b, 1, 0)
    for first, n in ((1, 1), (-1, 1), (0, 2), (2 ** 62, 1), (0, -1)):  # the last page is not full
        with pytest.raises(RuntimeError):
            pool.drop(b, first, n)
    pool.close(a)
    pool.close(b)
    assert pool.used == 0
    assert N.lib().kdn_page_pool_own(None, 0, 0, None, 0) == -1 and N.lib().kdn_page_pool_drop(None, 0, 0, 0) == -1


def make_pool(**kw):
    return HybridMemoryPool(6, 256, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device="cpu", anchor_layers=2, anchor_heads=2, **kw)


def test_a_slid_stream_keeps_its_positions():
    pool = make_pool(anchor_pages=40)
    s = pool.allocate_stream(0)
    pool.anchor_plan([s], [200])
    assert pool.anchor_slide([s], 50, 20) == 7  # pages 2 to 8 of 13: of the next token's window 151 is the first
    assert pool.anchor_tokens(s) == 200 - 7 * 16 and pool.anchor_pages_used == 6
    plan = pool.anchor_plan([s], [2])
    assert plan.positions.tolist() == [200, 201] and plan.context_lens.tolist() == [88] and plan.in_order
    assert pool.anchor_plan([s], [2], depths=[0, 1]).positions.tolist() == [202, 203]
    assert pool.anchor_slide([s], 50, 20) == 0 and pool.anchor_slide([s], 500) == 0
    f = pool.fork_stream(s)
    assert pool.anchor_plan([f], [1]).positions.tolist() == [202]
    with pytest.raises(ValueError):  # the window of a token at place 80 begins at 31, where freed pages were
        pool.anchor_truncate(f, 80)
    pool.anchor_truncate(f, 81)
    assert pool.anchor_plan([f], [1]).positions.tolist() == [193]
    with pytest.raises(ValueError):
        pool.anchor_slide([s], 0)
    with pytest.raises(ValueError):
        pool.anchor_evict([s], 10)
    with pytest.raises(ValueError):
        pool.anchor_weights(0)


def test_a_cut_stream_keeps_its_positions():
    pool = make_pool(anchor_pages=16, anchor_queries=8)
    s = pool.allocate_stream(0)
    plan = pool.anchor_plan([s], [100])
    assert plan.slots.tolist() == [s] and plan.run == 8 and plan.in_order
    f = pool.fork_stream(s)
    pool.anchor_evict([s, f], 100)
    assert pool.anchor_pages_used == 7
    pool.anchor_evict([f], 40, sinks=4, recent=8)
    assert pool.anchor_tokens(f) == 40 and pool.anchor_tokens(s) == 100 and pool.anchor_pages_used == 10
    plan = pool.anchor_plan([f, s], [1, 3])
    assert plan.positions.tolist() == [100, 100, 101, 102] and not plan.in_order and plan.slots.tolist() == [f, s]
    assert pool.anchor_plan([s], [9]).all_rows.numel() == 112  # more than run: the keys before it whole
    for back in (39, 1):  # into the places that are in no order
        with pytest.raises(ValueError):
            pool.anchor_truncate(f, back)
    pool.anchor_truncate(f, 40)
    assert pool.anchor_plan([f], [1]).positions.tolist() == [100]
    pool.anchor_truncate(f, 0)  # begins anew
    plan = pool.anchor_plan([f], [1])
    assert plan.in_order and plan.positions.tolist() == [0]
    for bad in (dict(streams=[s], keep=-1), dict(streams=[s], keep=4, sinks=-1), dict(streams=[s, s], keep=4)):
        with pytest.raises(ValueError):
            pool.anchor_evict(**bad)
    with pytest.raises(ValueError):
        pool.anchor_slide([s], 50)
    with pytest.raises(RuntimeError):
        pool.anchor_plan([s], [200])  # past the places
    assert pool.anchor_tokens(s) == 112
    forks = [pool.fork_stream(s) for _ in range(2)]
    with pytest.raises(RuntimeError):  # seven pages for each of the two, eight are free
        pool.anchor_evict(forks, 100)
    assert [pool.anchor_tokens(x) for x in forks] == [112, 112]
    with pytest.raises(ValueError):
        make_pool(anchor_queries=3)


@pytest.mark.parametrize("made", [False, True])
def test_a_pool_is_used_in_another_mode_than_it_was_made_in(made):
    with torch.inference_mode(made):
        pool = make_pool(anchor_pages=16, anchor_queries=8)
    with torch.inference_mode(not made):
        s = pool.allocate_stream(0)
        pool.anchor_plan([s], [30])
        f = pool.fork_stream(s)
        pool.anchor_evict([f], 20)
        pool.anchor_truncate(s, 10)
        assert [pool.anchor_tokens(x) for x in (s, f)] == [10, 20] and not pool.anchor_weights(1).any()


def test_layer_arguments():
    for bad in (dict(window=0), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            AnchorAttentionLayer(256, 4, 2, **bad)
    layer = AnchorAttentionLayer(256, 4, 2, window=8)
    pool = make_pool(anchor_pages=16, anchor_queries=4)
    s = pool.allocate_stream(0)
    pool.anchor_plan([s], [20])
    pool.anchor_evict([s], 10)
    with pytest.raises(ValueError, match="window"):
        layer.step(torch.zeros(1, 256), pool.anchor_plan([s], [1]), *pool.anchor_pages(0))
    plain = make_pool(anchor_pages=16)
    s = plain.allocate_stream(0)
    with pytest.raises(ValueError, match="no weights"):
        layer.step(torch.zeros(1, 256), plain.anchor_plan([s], [1]), *plain.anchor_pages(0), weights=pool.anchor_weights(0))


@pytest.mark.parametrize("seed", range(40))
def test_the_oracles_eviction(seed):
    """Against a sort of all places at once, and what a cut leaves of the tokens."""
    rng = random.Random(seed)
    L, gone, sinks, recent = rng.randint(1, 60), rng.randint(0, 50), rng.choice([0, 3]), rng.choice([0, 1, 10])
    settled, keep = rng.randint(0, L), rng.randint(0, L + 3)
    w = [rng.choice([0.0, 1.0, rng.random(), -1.0, float("nan"), float("inf")]) for _ in range(L)]
    pos = rng.sample(range(settled + gone), settled) + [-1] * (L - settled)
    moves, ww, pp = ob.evict(w, pos, L, keep, settled, gone, sinks, recent)
    at = [pos[j] if j < settled else j + gone for j in range(L)]
    n = min(L, keep)
    held = [at[j] < sinks or at[j] >= L + gone - recent for j in range(L)]  # whatever their weights
    order = sorted(range(L), key=lambda j: (at[j] >= sinks, not held[j], 0.0 if held[j] or not w[j] > 0 else -w[j], j))
    assert sorted(pp[:n]) == sorted(at[j] for j in order[:n])
    assert all(a >= n > b for a, b in moves) and len({b for _, b in moves}) == len(moves)
    by = {at[j]: w[j] for j in range(L)}
    assert all(ww[j] == by[pp[j]] or (ww[j] != ww[j] and by[pp[j]] != by[pp[j]]) for j in range(n))
    assert repr(ww[n:]) == repr(w[n:])


def test_the_oracles_window_and_weights():
    q, k, v = (torch.randn(9, h, 64, dtype=torch.float64) for h in (4, 2, 2))
    full, cut = (ob.attention(q, k, v, [0, 9], window=w, sinks=2)["y"] for w in (None, 9))
    assert torch.equal(full, cut) and torch.equal(full, oa.attention(q, k, v, [0, 9])["y"])
    seen = ob.visible(3, 2)(9, 9)
    assert seen[7].tolist() == [True, True, False, False, False, True, True, True, False] and seen[0].tolist() == [True] + [False] * 8
    r = ob.attention(q, k, v, [0, 9], window=3, sinks=2)
    w, = ob.weights(q, k, r["lse"], [0, 9], window=3, sinks=2)
    assert torch.allclose(w.sum(), torch.tensor(36.0, dtype=torch.float64))
    assert torch.allclose(w[0, 8], sum(torch.softmax((q[8, h] @ k[[0, 1, 6, 7, 8], 0].T) / 8, -1)[-1] for h in (0, 1)))
