"""The anchor layers' surface at its edges on the GPU: first calls in a capture, on another stream and in inference mode,
rows that no sequence has, layouts with odd strides, autograd's other modes, steps without tokens."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from kdn import _native as N
from kdn import anchor
from layers import AnchorAttentionLayer
from serving import HybridMemoryPool

DEV = "cuda:0"


def layer_and_input(**kw):
    torch.manual_seed(0)
    return AnchorAttentionLayer(256, 4, 2, rotary_dim=32, **kw).to(DEV), torch.randn(2, 40, 256, device=DEV)


@pytest.mark.gpu
def test_layer_first_called_on_two_streams():
    layer, x = layer_and_input()
    with torch.no_grad():
        want = AnchorAttentionLayer.forward(layer, x)
        torch.cuda.synchronize()
        again, _ = layer_and_input()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        out = []
        for s in (a, b):  # neither waits for the other
            with torch.cuda.stream(s):
                out.append(again(x))
        torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in out)


@pytest.mark.gpu
def test_layer_first_called_in_a_capture():
    layer, x = layer_and_input()
    with torch.no_grad():
        layer.w_q(x)  # the library's handles, which a capture cannot make
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(x)
        eager = layer(x)  # before the first replay
        torch.cuda.synchronize()
        other, _ = layer_and_input()
        assert torch.equal(eager, other(x))
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


@pytest.mark.gpu
def test_layer_trains_after_inference_mode():
    layer, x = layer_and_input()
    with torch.inference_mode():
        want = layer(x).clone()
    y = layer(x)
    assert torch.equal(y.detach(), want.clone())
    y.sum().backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in layer.parameters())


def odd_strides(t, single):
    """t as a view whose strides are no multiples of 16 bytes in the dimensions in `single`, each of one entry."""
    strides = list(t.contiguous().stride())
    for i in single:
        assert t.shape[i] == 1
        strides[i] = strides[i] + 8 * i + 1
    out = torch.as_strided(t.new_empty(4 * t.numel() + 64), t.shape, strides)
    out.copy_(t)
    assert out.stride() == tuple(strides)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,KV", [(1, 2), (5, 1), (1, 1)])
def test_strides_of_single_tokens_and_heads(n, KV, dtype):
    """A dimension of one entry has any stride, in every operator: its results are those of contiguous tensors."""
    d, P = 64, 16
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, dy = (torch.randn(n, h, d, generator=g, device=DEV).to(dtype) for h in (2 * KV, KV, KV, 2 * KV))
    odd = lambda t: odd_strides(t, [i for i in (0, 1) if t.shape[i] == 1])  # noqa: E731
    cu = torch.tensor([0, n], device=DEV)
    f = anchor.rotary_frequencies(d, device=DEV)[0]
    pos = torch.arange(n, device=DEV)
    for a, b in zip(anchor.rotary(odd(q), odd(k), pos, f), anchor.rotary(q, k, pos, f)):
        assert torch.equal(a, b)
    want, got = [], []
    for out, change in ((want, lambda t: t.clone()), (got, odd)):
        leaves = [change(t).requires_grad_(True) for t in (q, k, v)]
        y = anchor.attention(*leaves, cu)
        out += [y.detach(), *torch.autograd.grad(y, leaves, change(dy))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = odd(torch.zeros_like(q))
    anchor.attention(q, k, v, cu, out=held)
    assert torch.equal(held, want[0])
    turned = odd(q)
    anchor.rotary(turned, None, pos, f, in_place=True)
    assert torch.equal(turned, anchor.rotary(q, None, pos, f)[0])
    pages = [torch.zeros(1, KV, P, d, dtype=dtype, device=DEV) for _ in range(4)]
    pages[2:] = [odd_strides(t, [i for i in (0, 1) if t.shape[i] == 1]) for t in pages[2:]]
    anchor.page_append(k, v, pages[0], pages[1], pos)
    anchor.page_append(odd(k), odd(v), pages[2], pages[3], pos)
    assert torch.equal(pages[0], pages[2]) and torch.equal(pages[1], pages[3])
    table, ctx = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    want = anchor.tree_attention(q, k, v, *pages[:2], table, ctx, cu)
    wide = torch.zeros(1, 9, dtype=torch.int32, device=DEV).t()[3:4]  # one page number, strides (1, 9)
    assert torch.equal(anchor.tree_attention(odd(q), odd(k), odd(v), *pages[2:], wide, ctx, cu, out=odd(torch.zeros_like(q))), want)


@pytest.mark.gpu
def test_tokens_further_apart_than_a_copy_reaches():
    """Two tokens 2^25 elements apart (a copy of 64 such rows would pass 32-bit offsets): copied first, as other layouts are."""
    far = torch.zeros(2**25 + 256, dtype=torch.float32, device=DEV)
    q = torch.randn(2, 2, 64, device=DEV)
    view = torch.as_strided(far, (2, 2, 64), (2**25, 64, 1))
    view.copy_(q)
    cu = torch.tensor([0, 2], device=DEV)
    assert torch.equal(anchor.attention(view, view, view, cu), anchor.attention(q, q, q, cu))


def step_of(lens, new, pad, lead=0, H=8, KV=2, d=64, dtype=torch.bfloat16):
    """A step's tensors with `lead` rows before the first stream's and `pad` behind the last's, the pages in order."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n, P = lead + sum(new) + pad, 16
    q, k, v = (torch.randn(n, h, d, generator=g, device=DEV).to(dtype) for h in (H, KV, KV))
    per = max([1, *(-(-x // P) for x in lens)])
    kp, vp = (torch.randn(max(1, len(lens)) * per, KV, P, d, generator=g, device=DEV).to(dtype) for _ in range(2))
    table = torch.arange(len(lens) * per, dtype=torch.int32, device=DEV).view(len(lens), per)
    cu = torch.tensor([lead, *new], device=DEV).cumsum(0)
    return q, k, v, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=DEV), cu


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,new,pad,lead", [([700, 20], [1, 1], 37, 0), ([700, 20], [1, 1], 0, 3), ([300, 0, 7], [20, 0, 33], 5, 2),
                                               ([40] * 70, [1] * 70, 442, 0), ([50, 60], [0, 0], 9, 0)])
def test_rows_that_no_stream_has_are_zeros(lens, new, pad, lead, d, dtype):
    step = step_of(lens, new, pad, lead, d=d, dtype=dtype)
    n, inside = step[0].shape[0], slice(lead, lead + sum(new))
    want = anchor.tree_attention(*(t[inside] for t in step[:3]), *step[3:7], step[7] - lead)
    for held in (torch.full_like(step[0], float("nan")), torch.full((n, 10, d), 7.0, dtype=dtype, device=DEV)[:, 1:9]):
        y = anchor.tree_attention(*step, out=held)
        assert torch.equal(y[inside], want)
        assert not y[:lead].any() and not y[lead + sum(new):].any()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [4, 16])
def test_tokens_past_max_new_are_zeros(H):
    new = [5, 1, 3, 70, 0, 2]
    step = step_of([30, 300, 0, 16, 3, 40], new, 4, H=H)
    y = anchor.tree_attention(*step, max_new=3, out=torch.full_like(step[0], float("nan")))
    own = torch.cat([torch.arange(n) < 3 for n in [*new]] + [torch.zeros(4, dtype=torch.bool)]).to(DEV)
    assert not y[~own].any()
    cut = [min(n, 3) for n in new]
    want = anchor.tree_attention(*(t[own] for t in step[:3]), *step[3:7], torch.tensor([0, *cut], device=DEV).cumsum(0), max_new=3)
    assert torch.equal(y[own], want)
    y = anchor.tree_attention(*step, out=torch.full_like(step[0], float("nan")))  # 64 of the 70
    assert torch.isfinite(y).all() and not y[9 + 64:9 + 70].any() and y[9 + 63].any()


@pytest.mark.gpu
def test_a_padded_step_without_streams_is_zeros():
    q, k, v, kp, vp, table, ctx, cu = step_of([], [], 6)
    y = anchor.tree_attention(q, k, v, kp, vp, table.view(0, 1), ctx, cu, out=torch.full_like(q, float("nan")))
    assert not y.any()


@pytest.mark.gpu
def test_a_call_without_streams_needs_y_alone():
    y = torch.full((6, 8, 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    a = N.TreeAttnArgs()
    a.total_new, a.max_new, a.max_context, a.H, a.H_kv, a.d, a.dtype, a.scale = 6, 1, 4096, 8, 2, 64, N.KDN_DTYPE_BF16, 0.125
    a.page_tokens, a.num_pages, a.table_width, a.table_stride, a.y = 16, 1, 256, 256, y.data_ptr()
    a.y_stride[0], a.y_stride[1] = 512, 64
    assert N.lib().kdn_tree_attn(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    assert not y.any()


@pytest.mark.gpu
def test_a_padded_step_in_a_graph():
    """A step captured for eight streams' tokens, replayed with fewer of them."""
    step = step_of([300, 20, 77, 1, 50, 60, 70, 5], [1] * 8, 0)
    g = torch.cuda.CUDAGraph()
    anchor.tree_attention(*step, max_new=1)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = anchor.tree_attention(*step, max_new=1)
    for live in (8, 5, 2, 7):
        step[7].copy_(torch.arange(9, device=DEV).clamp(max=live))
        g.replay()
        torch.cuda.synchronize()
        want = anchor.tree_attention(*(t[:live] for t in step[:3]), *step[3:5], step[5][:live], step[6][:live], torch.arange(live + 1, device=DEV),
                                     max_new=1, max_context=step[5].shape[1] * 16)
        assert not y[live:].any()
        assert float((y[:live].float() - want.float()).abs().max()) < 2.0 ** -6  # chunks of another length: their sums' order


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lead,lead_k,lens,pad,pad_k,H,KV", [(5, 5, [70, 0, 33], 4, 4, 4, 2), (0, 200, [40, 130], 0, 3, 4, 1), (140, 0, [1, 129], 7, 0, 8, 8),
                                                             (3, 9, [7] * 62, 5, 6, 4, 2), (3, 9, [7] * 63, 5, 6, 4, 2), (40, 150, [3] * 150, 33, 0, 4, 4),
                                                             (600, 700, [2100], 300, 10, 32, 8), (9, 9, [], 0, 0, 4, 2), (260, 260, [4500], 0, 0, 32, 8)])
def test_rows_outside_the_offsets(lead, lead_k, lens, pad, pad_k, H, KV, d, dtype):
    """Rows before the first offset and behind the last: zeros, with lse -infinity and zero gradients, whatever is in memory;
    the sequences are what they are without them."""
    g = torch.Generator(device=DEV).manual_seed(2)
    n = sum(lens)
    q, k, v, dy = (torch.randn(x, h, d, generator=g, device=DEV).to(dtype) for x, h in
                   ((lead + n + pad, H), (lead_k + n + pad_k, KV), (lead_k + n + pad_k, KV), (lead + n + pad, H)))
    cu = torch.tensor([0, *lens], device=DEV).cumsum(0)
    iq, ik = slice(lead, lead + n), slice(lead_k, lead_k + n)
    nan = [torch.full((8 * max(q.numel(), 1024),), float("nan"), device=DEV)]
    nan.clear()  # what the outputs and the workspace are likely made of
    y, lse, low = anchor.attention_forward(q, k, v, cu + lead, cu + lead_k, out=torch.full_like(q, float("nan")), return_lse=True, return_low=True)
    grads = anchor.attention_backward(q, k, v, y, lse, dy, cu + lead, cu + lead_k, low=low)
    for t, i in ((y, iq), (grads[0], iq), (grads[1], ik), (grads[2], ik)):
        assert not t[:i.start].any() and not t[i.stop:].any()
    assert torch.isneginf(lse[:, :lead]).all() and torch.isneginf(lse[:, lead + n:]).all()
    y2, lse2, low2 = anchor.attention_forward(q[iq], k[ik], v[ik], cu, return_lse=True, return_low=True)
    want = [y2, *anchor.attention_backward(q[iq], k[ik], v[ik], y2, lse2, dy[iq], cu, low=low2)]
    # another split of a row's keys or of a key's rows: fp32 sums in another order, then the rounding
    for t, w in zip([y[iq], grads[0][iq], grads[1][ik], grads[2][ik]], want):
        scale = float(w.float().norm()) + 1e-30
        assert float((t.float() - w.float()).norm()) <= (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18) * scale


@pytest.mark.gpu
def test_serving_operators_do_not_drop_gradients():
    """As the ragged steps: the attention's output raises on backward; what goes into the pages is refused."""
    q, k, v, kp, vp, table, ctx, cu = step_of([30, 0], [1, 2], 0)
    want = anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu)
    for i in range(5):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v, kp, vp))]
        y = anchor.tree_attention(*args, table, ctx, cu)
        assert torch.equal(y.detach(), want)
        with pytest.raises(NotImplementedError, match="tree_attention"):
            y.sum().backward()
        with torch.no_grad():
            assert not anchor.tree_attention(*args, table, ctx, cu).requires_grad
    rows = torch.tensor([30, 32, 33], device=DEV)
    for i in (0, 1):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((k, v))]
        with pytest.raises(ValueError):
            anchor.page_append(*args, kp, vp, rows)
        with torch.no_grad():
            anchor.page_append(*args, kp, vp, rows)


@pytest.mark.gpu
def test_second_derivatives():
    """Of the attention they are refused; the rotation's are exact: with q' = R q, |dL/dq|^2 for L = |q'|^2 / 2 and a magnitude m
    is m^4 |q|^2, whose derivative is 2 m^4 q."""
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k = (torch.randn(9, h, 64, generator=g, device=DEV).requires_grad_(True) for h in (4, 2))
    f = anchor.rotary_frequencies(64, device=DEV)[0]
    pos, cu = torch.arange(9, device=DEV), torch.tensor([0, 9], device=DEV)
    for keys in (k, None):
        a, b = anchor.rotary(q, keys, pos, f, magnitude=1.25)
        loss = (a * a).sum() / 2 + (0 if keys is None else (b * b).sum() / 2)
        leaves = [q] if keys is None else [q, k]
        first = torch.autograd.grad(loss, leaves, create_graph=True)
        second = torch.autograd.grad(sum((t * t).sum() for t in first), leaves)
        for x, d in zip(leaves, second):
            want = 2 * 1.25 ** 4 * x.detach()  # four turns, each within 8 units of 2^-24 of |a| + |b|
            assert float((d - want).abs().max()) < 4 * 8 * 2.0 ** -24 * 2 * float(want.abs().max())
    y = anchor.attention(q, k, k, cu)
    dq, = torch.autograd.grad((y * y).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dq * dq).sum().backward()


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is not lost: every operator that computes raises, with gradients enabled or not."""
    q, k, v, kp, vp, table, ctx, cu = step_of([30, 0], [1, 2], 0, dtype=torch.float32)
    f, pos = anchor.rotary_frequencies(64, device=DEV)[0], torch.arange(3, device=DEV)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for calls in ((lambda: anchor.rotary(dual(q), k, pos, f), lambda: anchor.rotary(q, dual(k), pos, f), lambda: anchor.rotary(dual(q), None, pos, f)),
                      [lambda i=i: anchor.attention(*(dual(t) if i == j else t for j, t in enumerate((q, k, v))), cu) for i in range(3)],
                      [lambda i=i: anchor.tree_attention(*(dual(t) if i == j else t for j, t in enumerate((q, k, v, kp, vp))), table, ctx, cu)
                       for i in range(5)]):
            for call in calls:
                with pytest.raises(NotImplementedError):
                    call()
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    call()
        with pytest.raises(ValueError):
            anchor.page_append(dual(k), v, kp, vp, pos)
        plain = anchor.attention(q, k, v, cu)  # nothing of it has a tangent
    assert torch.equal(plain, anchor.attention(q, k, v, cu))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing_to_do(dtype):
    """Steps of no tokens or no streams, and empty batches: outputs of their shape, and gradients of zero."""
    layer = AnchorAttentionLayer(256, 4, 2).to(DEV, dtype)
    pool = HybridMemoryPool(4, 64, num_layers=1, num_heads=1, val_dim=16, lifted_dim=64, device=DEV, anchor_layers=1, anchor_heads=2,
                            anchor_pages=16, anchor_dtype=dtype)
    some = [pool.allocate_stream(0) for _ in range(2)]
    layer.step(torch.randn(21, 256, device=DEV).to(dtype), pool.anchor_plan(some, [20, 1]), *pool.anchor_pages(0))
    x = torch.zeros(0, 256, dtype=dtype, device=DEV)
    for streams in (some, []):
        none = [0] * len(streams)
        assert layer.step(x, pool.anchor_plan(streams, none), *pool.anchor_pages(0)).shape == (0, 256)
        out, k, v = layer.step(x, pool.anchor_plan(streams, none, depths=[]), *pool.anchor_pages(0))
        assert out.shape == (0, 256) and k.shape == v.shape == (0, 2, 64)
    for shape, cu in (((0, 7, 256), None), ((3, 0, 256), None), ((0, 256), torch.tensor([0, 0, 0], device=DEV)), ((0, 256), torch.tensor([0], device=DEV))):
        layer.zero_grad()
        x = torch.zeros(shape, dtype=dtype, device=DEV, requires_grad=True)
        y = layer(x, cu)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and not any(p.grad.any() for p in layer.parameters())
    q = torch.zeros(0, 4, 64, dtype=dtype, device=DEV)
    assert anchor.tree_attention(q, q, q, *(torch.zeros(1, 4, 16, 64, dtype=dtype, device=DEV),) * 2, torch.zeros(0, 1, dtype=torch.int32, device=DEV),
                                 torch.zeros(0, dtype=torch.int32, device=DEV)).shape == q.shape


@pytest.mark.gpu
def test_writes_in_place_are_seen_by_autograd():
    """A tensor that a backward saved and an operator then wrote: the backward refuses it, as after torch's own writes."""
    q, k, v, kp, vp, table, ctx, cu = step_of([30, 0], [1, 2], 0, dtype=torch.float32)
    f, pos = anchor.rotary_frequencies(64, device=DEV)[0], torch.arange(3, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    for write in (lambda t: anchor.rotary(t, None, pos, f, in_place=True), lambda t: anchor.rotary(k.clone().repeat(1, 4, 1), t, pos, f, in_place=True),
                  lambda t: anchor.attention(q, k, v, cu, out=t), lambda t: anchor.tree_attention(q, k, v, kp, vp, table, ctx, cu, out=t)):
        held = q.clone()
        loss = (held * w).sum()
        with torch.no_grad():
            write(held)
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
    with torch.inference_mode():
        held = q.clone()
        anchor.rotary(held, None, pos, f, in_place=True)
    assert torch.equal(held, anchor.rotary(q, None, pos, f)[0])
