"""The anchor layers' surface at its edges, with no GPU: the layer's frequencies, a plan's arguments, the operators' checks."""
import ctypes
import subprocess
import sys

import numpy as np
import pytest
import torch

from kdn import _native as N
from kdn import anchor
from layers import AnchorAttentionLayer
from serving import HybridMemoryPool


def test_frequencies_are_made_with_the_layer():
    """They are there before the first call, normal tensors whichever mode that call is in (training saves them), and float64
    whatever the layer is cast to."""
    layer = AnchorAttentionLayer(128, 2, 1, rotary_dim=32)
    with torch.inference_mode():
        first = layer.inv_freq(torch.device("cpu"))
    assert not first.is_inference()
    want = 10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    for cast in (layer, layer.to(torch.bfloat16), layer.double()):
        f = cast.inv_freq(torch.device("cpu"))
        assert f.dtype == torch.float64 and float((f - want).abs().max()) < 1e-15
    with torch.inference_mode():
        assert not AnchorAttentionLayer(128, 2).inv_freq(torch.device("cpu")).is_inference()


def test_frequencies_follow_the_parameters():
    with torch.device("meta"):
        layer = AnchorAttentionLayer(128, 2, 1, rotary_dim=32)
    assert layer.inv_freq(torch.device("meta")).device.type == "meta"
    layer.to_empty(device="cpu")
    f = layer._inv_freq
    assert f.device.type == "cpu" and float(f[0]) == 1.0
    assert layer.inv_freq(torch.device("cpu")) is f
    assert "inv_freq" not in "".join(layer.state_dict())
    for name in ("w_q", "w_k", "w_v", "w_out"):  # projections of another kind, without parameters of their own
        setattr(layer, name, torch.nn.Identity())
    assert layer.to("cpu")._inv_freq is f
    layer.w_q = torch.nn.Linear(4, 4, device="meta")
    assert layer.to(torch.float64)._inv_freq.device.type == "meta"


def pool_of(*lens, pages=8):
    """A host pool (bookkeeping alone) whose streams have `lens` tokens."""
    pool = HybridMemoryPool(4, 64, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device="cpu", anchor_layers=1, anchor_heads=1,
                            anchor_pages=pages)
    streams = [pool.allocate_stream(n) for n in lens]
    pool.anchor_plan(streams, list(lens))
    return pool, streams


@pytest.mark.parametrize("depths", [[0], [0, 1], [0, 1, 1, 2], [], [[0, 1, 2]], 0, [0.0, 1.0, 2.0], torch.tensor([0, 1]), torch.zeros(3, 1, dtype=torch.int64)])
def test_a_plan_of_drafts_has_a_depth_for_each(depths):
    pool, (s,) = pool_of(20)
    with pytest.raises(ValueError):
        pool.anchor_plan([s], [3], depths=depths)
    for good in ([0, 1, 1], (0, 1, 1), torch.tensor([0, 1, 1]), torch.tensor([0, 1, 1], dtype=torch.int16)):
        assert pool.anchor_plan([s], [3], depths=good).positions.tolist() == [20, 21, 21]
    assert pool.anchor_tokens(s) == 20


@pytest.mark.parametrize("new", [[5], [5, 1, 1], []])
@pytest.mark.parametrize("drafts", [False, True])
def test_a_plan_has_a_number_of_tokens_for_each_stream(new, drafts):
    pool, streams = pool_of(20, 3)
    with pytest.raises(ValueError):
        pool.anchor_plan(streams, new, depths=[0] * sum(new) if drafts else None)
    assert [pool.anchor_tokens(s) for s in streams] == [20, 3]


@pytest.mark.parametrize("bad,error", [(1.0, TypeError), ("1", TypeError), (None, TypeError), (-1, ValueError)])
def test_a_refused_plan_changes_no_stream(bad, error):
    pool, streams = pool_of(20, 3)
    with pytest.raises(error):
        pool.anchor_plan(streams, [5, bad])
    assert [pool.anchor_tokens(s) for s in streams] == [20, 3] and pool.anchor_pages_used == 3
    plan = pool.anchor_plan(streams, np.array([5, 1]))  # whole numbers of any kind
    assert plan.positions.tolist() == [20, 21, 22, 23, 24, 3] and plan.max_new == 5
    assert pool.anchor_plan(streams, torch.tensor([1, 2])).positions.tolist() == [25, 4, 5]


def test_a_pool_that_lives_to_the_end():
    """Destroyed while the interpreter takes its modules apart: nothing is printed."""
    path = anchor.__file__.rsplit("kdn", 1)[0]
    code = f"import sys; sys.path.insert(0, {path!r}); from kdn import anchor; pool = anchor.PagePool(4, 16, 2); pool.open()"
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "PagePool" not in done.stderr, done.stderr


def test_plans_without_tokens():
    pool, streams = pool_of(20, 3)
    for plan in (pool.anchor_plan(streams, [0, 0]), pool.anchor_plan(streams, [0, 0], depths=[])):
        assert plan.max_new == 0 and plan.positions.tolist() == [] and plan.cu_seqlens.tolist() == [0, 0, 0] and plan.context_lens.tolist() == [20, 3]
    for plan in (pool.anchor_plan([], []), pool.anchor_plan([], [], depths=[])):
        assert plan.max_new == 0 and plan.positions.tolist() == [] and plan.cu_seqlens.tolist() == [0] and plan.page_table.shape[0] == 0
    assert pool.anchor_plan(streams, [0, 1]).positions.tolist() == [3]


def test_a_call_without_new_tokens_needs_no_bound():
    a = N.TreeAttnArgs()
    a.num_seqs, a.H, a.H_kv, a.d, a.dtype, a.scale, a.page_tokens = 2, 8, 2, 128, 1, 0.1, 16
    assert N.lib().kdn_tree_attn(ctypes.byref(a), None) == 0 and N.lib().kdn_tree_attn_workspace_bytes(ctypes.byref(a)) > 0
    a.total_new = 1
    assert N.lib().kdn_tree_attn(ctypes.byref(a), None) == -1 and N.lib().kdn_tree_attn_workspace_bytes(ctypes.byref(a)) == 0


def test_errors_name_what_the_anchor_layers_support():
    for status, words in ((-2, ("d 64 or 128", "64 new tokens", "pages", "d_k must be 64")), (-6, ("slot", "stream", "page"))):
        text = N.lib().kdn_strerror(status).decode()
        assert all(w in text for w in words), text
    pool = anchor.PagePool(1, 16, 1)
    s = pool.open()
    with pytest.raises(RuntimeError, match="page"):
        pool.extend(s, 17)


def test_sizes_past_what_the_grid_takes():
    """Refused from the numbers alone, however large: no product of them wraps into one that passes."""
    def args(**kw):
        a = N.TreeAttnArgs()
        a.num_seqs, a.total_new, a.max_new, a.max_context, a.H, a.H_kv, a.d, a.dtype, a.scale = 2, 2, 1, 4096, 8, 2, 128, 1, 0.1
        a.page_tokens, a.num_pages, a.table_width, a.table_stride = 16, 999, 256, 256
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    size, call = N.lib().kdn_tree_attn_workspace_bytes, N.lib().kdn_tree_attn
    big = 1 << 20
    for bad in (dict(page_tokens=1 << 31, table_width=1), dict(page_tokens=1 << 32, table_width=1), dict(page_tokens=1 << 62, table_width=1),
                dict(num_seqs=(1 << 31) - 1, H=big, H_kv=big, max_context=1 << 30, table_width=1 << 26),
                dict(num_seqs=1 << 30, H=big, H_kv=big, max_context=1 << 25, table_width=1 << 21),
                dict(num_seqs=1 << 30, H=big, H_kv=1, max_new=64), dict(num_seqs=1 << 20, H=big, H_kv=1, max_new=64)):
        assert size(args(**bad)) == 0 and call(args(**bad), None) == -2, bad
    for bad in (dict(table_width=255), dict(max_context=4097)):
        assert size(args(**bad)) == 0 and call(args(**bad), None) == -1, bad
    # a wide table of small pages, and one page of a whole context
    assert size(args(table_width=1 << 60)) == size(args(page_tokens=1 << 30, table_width=1)) == size(args()) > 16


@pytest.mark.parametrize("bad", [torch.tensor([[0, 1 << 32]]), [(0, (1 << 32) + 1)], torch.tensor([[0, 2, 4], [1, 3, 5]]), [(0.0, 1.5)],
                                 torch.tensor([[[0, 1]]]), torch.tensor([[True, False]])])
def test_page_numbers_are_not_cut(bad):
    """Numbers past 32 bits, fractions and lists of another shape name no pages: refused, not wrapped or cut into others."""
    with pytest.raises(ValueError):
        anchor._pairs(bad)


@pytest.mark.parametrize("good", [[(0, 1), (2, 3)], torch.tensor([[0, 1], [2, 3]]), torch.tensor([[0, 2], [1, 3]], dtype=torch.int32).t(), np.array([[0, 1], [2, 3]]),
                                  [0, 1, 2, 3]])
def test_page_pairs_of_any_whole_numbers(good):
    p = anchor._pairs(good)
    assert p.dtype == torch.int32 and p.is_contiguous() and p.tolist() == [[0, 1], [2, 3]]
    assert anchor._pairs([]).shape == (0, 2)
