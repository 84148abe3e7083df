"""Operators of bounded contexts (include/kdn_bounded.h): what keeps an anchor layer's cache from growing with a stream's whole
past, next to recurrent states of fixed size.

    attention_weights   the weight that each key of a batch of prompts got from all rows, or from the last ones
    evict               of each stream, layer and head the keys of least weight give way; the kept ones close up

Decode steps add to the same weights in their own pass (`anchor.tree_attention(weights=)`).  The other way to bound a context is
a sliding window with sinks: `window` and `sinks` of `anchor.attention` and `anchor.tree_attention`.

torch supplies device memory and the current HIP stream; every computation is a HIP kernel in libkdn.so; nothing here waits for
the device.  The reference never bounds its anchor pages (serving/hybrid_memory_pool.{h,cpp}).
"""
from __future__ import annotations

import functools
import operator
import struct
from typing import Optional

import torch

from . import _native as N
from .anchor import _BF16, _F32, _device, _heads, _ints, _key_weights, _raw_stream, _scale, _steps, _tracked, _window
from .ops import _tag, require_device

# The argument structs of include/kdn_bounded.h as packed bytes (tests/test_bounded_host.py holds them against the mirrors).
_WEIGHTS = struct.Struct("@qqqqqiiifqqPP" + 2 * "Pqq" + "P" + "Pqq" + "qqPPN")
_EVICT = struct.Struct("@qqqiiqqqqqqq" + 6 * "P" + 2 * "Pqqqq" + 2 * "Pqqq" + "qqPN")


@functools.lru_cache(maxsize=64)
def _weights_bytes(nseq: int, nq: int, nk: int, H: int, KV: int, d: int, dtype: int, window: int, sinks: int) -> int:
    """kdn_attn_weights_workspace_bytes, which reads sizes only (each sequence has a slot)."""
    return N.lib().kdn_attn_weights_workspace_bytes(_WEIGHTS.pack(nseq, nq, nk, H, KV, d, dtype, 0, 1.0, window, sinks, 4, 4, *(0,) * 10, 0, nseq, 0, 0, 0))


def attention_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, weights: torch.Tensor, cu_seqlens: torch.Tensor,
                      cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None, window: Optional[int] = None,
                      sinks: int = 0, add: bool = False, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """weights[b, e, j] = the softmax weight that key j of sequence b got from all its query rows and the query heads of key
    head e, written where it is; weights.

    q (tokens, H, d), k (tokens, H_kv, d), cu_seqlens, cu_seqlens_k, scale, window and sinks as `anchor.attention` takes them, lse
    (H, tokens) float32 as `anchor.attention_forward(..., return_lse=True)` gave it for these rows (or for more of them: the last rows of
    each sequence alone, q's and lse's, say what the end of a prompt looks at).  weights (slots, H_kv, places) float32, places next to
    one another.  `add`: keys before a sequence's first row here (a prompt's earlier pieces) are added to, the others set; else
    all of a sequence's keys are set.  Keys past `places` are skipped; places behind a sequence's keys stay.  `slots` (sequences,):
    which row is a sequence's (none given: its number), no two the same; of those out of range nothing is written.  Not
    differentiable."""
    what = "attention_weights"
    if _tracked(q, k, lse):
        raise ValueError(f"{what}: the weights have no gradient; call it under torch.no_grad() or detach q, k and lse")
    qs, ks = _heads(q, f"{what} q"), _heads(k, f"{what} k", q)
    n, H, d = q.shape
    KV, dev = k.shape[1], q.get_device()
    if KV == 0 or H == 0 or H % KV:
        raise ValueError(f"{what}: q has a multiple of k's heads; got q {tuple(q.shape)}, k {tuple(k.shape)}")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or (cu_seqlens_k is not None and cu_seqlens_k.shape != cu_seqlens.shape):
        raise ValueError(f"{what}: cu_seqlens are (sequences + 1,), the same number for queries and keys")
    if cu_seqlens_k is None and k.shape[0] != n:
        raise ValueError(f"{what}: {n} queries and {k.shape[0]} keys need cu_seqlens_k")
    if tuple(lse.shape) != (H, n) or lse.dtype is not _F32 or lse.device != q.device:
        raise ValueError(f"{what}: lse is ({H}, {n}) float32 on {q.device}, got {tuple(lse.shape)} {lse.dtype} on {lse.device}")
    cu_q = _ints(cu_seqlens, f"{what} cu_seqlens", torch.int64, dev)
    cu_k = None if cu_seqlens_k is None else _ints(cu_seqlens_k, f"{what} cu_seqlens_k", torch.int64, dev)
    near, first = _window(window, sinks, what)
    B = cu_q.shape[0] - 1
    slots, slots_at = _key_weights(weights, slots, B, (KV,), q, what)
    lse = lse.contiguous()
    tag, s0, s1, _ = _tag(q.dtype, what), *weights.stride()
    torch.autograd.graph.increment_version(weights)
    with _device(dev):
        nbytes = _weights_bytes(B, n, k.shape[0], H, KV, d, tag, near, first)
        ws = q.new_empty(nbytes, dtype=torch.uint8)
        N.check(N.lib().kdn_attn_weights(_WEIGHTS.pack(B, n, k.shape[0], H, KV, d, tag, bool(add), _scale(scale, d, what), near, first, cu_q.data_ptr(),
                                                       0 if cu_k is None else cu_k.data_ptr(), *qs[1:], *ks[1:], lse.data_ptr(), weights.data_ptr(),
                                                       s0, s1, weights.shape[2], weights.shape[0], slots_at, ws.data_ptr(), nbytes),
                                         _raw_stream(dev)), "kdn_attn_weights")
    return weights


def _layers(t: torch.Tensor, what: str):
    """A cache's pages (pages, layers, heads, page_tokens, d), or of one layer without that dimension: (its address, the page, layer,
    head and token strides); used where it is, never copied."""
    if not t.is_cuda:
        require_device(t, what)
    dim, dt = t.dim(), t.dtype
    if dim not in (4, 5) or t.shape[-1] not in (64, 128) or (dt is not _BF16 and dt is not _F32):
        raise ValueError(f"{what}: expects (pages, layers, heads, page_tokens, d), or without layers, of bfloat16 or float32 and d = 64 or 128; "
                         f"got {tuple(t.shape)} {dt}")
    a, *rest, last = t.stride()
    steps = (a, 0, *rest) if dim == 4 else (a, *rest)
    p, odd = t.data_ptr(), 7 if dt is _BF16 else 3
    if (steps[0] | steps[1] | steps[2] | steps[3]) & odd:
        steps = _steps(t)
        steps = (steps[0], 0, *steps[1:]) if dim == 4 else steps
    if last != 1 or p & 15 or (steps[0] | steps[1] | steps[2] | steps[3]) & odd:
        raise ValueError(f"{what}: needs contiguous rows that start on 16 bytes (a cache is used where it is, never copied)")
    if 0 in rest or a == 0:
        if any(x == 0 and n > 1 for x, n in zip((a, *rest), t.shape)):
            raise ValueError(f"{what}: rows are written where they are, and these lie on one another (an expanded tensor)")
    return p, *steps


@functools.lru_cache(maxsize=64)
def _evict_bytes(*sizes) -> int:
    """kdn_evict_workspace_bytes, which reads sizes and whether there are slots only."""
    streams, layers, heads, d, dtype, page_tokens, pages, width, max_len, slots, places, rows = sizes
    return N.lib().kdn_evict_workspace_bytes(_EVICT.pack(streams, layers, heads, d, dtype, page_tokens, pages, width, 0, max_len, 0, 0, *(0,) * 5,
                                                         4 if slots else 0, *(0,) * 18, places, rows, 0, 0))


def evict(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, keep: torch.Tensor,
          weights: torch.Tensor, positions: torch.Tensor, settled: Optional[torch.Tensor] = None, evicted: Optional[torch.Tensor] = None,
          sinks: int = 0, recent: int = 0, slots: Optional[torch.Tensor] = None, max_len: Optional[int] = None) -> None:
    """Cuts each stream's cache from lens[b] places to min(lens[b], keep[b]), of each layer and key head on its own, in place.

    k_pages, v_pages (pages, layers, H_kv, page_tokens, d) in any strides (or of one layer, without that dimension), page_table
    (streams, width) int32, lens and keep (streams,) on the device.  weights (slots, layers, H_kv, places) float32 and positions,
    the same in int32 (without layers if the pages have none): place j of a stream has the token at position positions[..., j] if
    j < settled[b] (none given: 0), else j + evicted[b] (0; how many of a stream's tokens have no place any more).

    What stays: the positions below `sinks`, then the last `recent` of the stream's, then those of largest weight (one that is
    no positive number counts as 0), of equals the lowest places.  That goes for the last `recent`, too: with a `recent` of at most
    keep - sinks all of them stay, with a larger one the latest may be those that go.  The kept places behind the new length go, in order, to the
    given-up ones before it, in order, with key, value, weight and position; attention does not ask for an order of its keys.
    Afterwards positions of all places below the new length are there: settled is then the new length, evicted greater by what
    went.  What lies behind stays as it is.  The pages of places below the new length have to be the stream's own
    (`PagePool.own`), slots and pages distinct.  `slots` as in `attention_weights`; `max_len` (what page_table holds and there are places
    for) bounds lens from the host, longer ones are cut to it: nothing is read back."""
    if _tracked(k_pages, v_pages, weights):
        raise ValueError("evict: the pages have no gradient; call it under torch.no_grad()")
    kp, vp = _layers(k_pages, "evict k_pages"), _layers(v_pages, "evict v_pages")
    shape, dev, dt = k_pages.shape, k_pages.get_device(), k_pages.dtype
    plain = len(shape) == 4
    pages, P, d = shape[0], shape[-2], shape[-1]
    heads = shape[1:2] if plain else shape[1:3]
    if v_pages.shape != shape or v_pages.dtype is not dt or v_pages.get_device() != dev:
        raise ValueError(f"evict: pages {tuple(shape)} {dt} and {tuple(v_pages.shape)} {v_pages.dtype} differ")
    if page_table.get_device() != dev or page_table.dim() != 2 or page_table.dtype is not torch.int32 or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"evict: page_table is (streams, width) int32 on {k_pages.device}, got {tuple(page_table.shape)} {page_table.dtype} "
                         f"on {page_table.device}")
    B, width = page_table.shape
    slots, slots_at = _key_weights(weights, slots, B, heads, k_pages, "evict")
    rows, places = weights.shape[0], weights.shape[-1]
    if positions.shape != weights.shape or positions.dtype is not torch.int32 or positions.get_device() != dev or \
            (places > 1 and positions.stride(-1) != 1) or any(s == 0 and n > 1 for s, n in zip(positions.stride(), positions.shape)):
        raise ValueError(f"evict: positions are {tuple(weights.shape)} int32 on {weights.device}, places next to one another and none twice; got "
                         f"{tuple(positions.shape)} {positions.dtype} on {positions.device}")
    lens, keep = _ints(lens, "evict lens", torch.int32, dev, B), _ints(keep, "evict keep", torch.int32, dev, B)
    settled = None if settled is None else _ints(settled, "evict settled", torch.int32, dev, B)
    evicted = None if evicted is None else _ints(evicted, "evict evicted", torch.int32, dev, B)
    sinks, recent = operator.index(sinks), operator.index(recent)
    if sinks < 0 or recent < 0:
        raise ValueError(f"evict: sinks and recent are 0 or more, got {sinks}, {recent}")
    most = min(width * P, places)
    if max_len is not None:
        most = min(operator.index(max_len), most)
        if most < 0:
            raise ValueError(f"evict: max_len is 0 or more, got {max_len}")
    w0, *w1 = weights.stride()
    p0, *p1 = positions.stride()
    layers, KV = (1, *heads) if plain else heads
    torch.autograd.graph.increment_version((k_pages, v_pages, weights, positions))
    with _device(dev):
        nbytes = _evict_bytes(B, layers, KV, d, _tag(dt, "evict"), P, pages, width, most, slots_at != 0, places, rows)
        ws = weights.new_empty(nbytes, dtype=torch.uint8)
        N.check(N.lib().kdn_evict(_EVICT.pack(B, layers, KV, d, _tag(dt, "evict"), P, pages, width, page_table.stride(0), most, min(sinks, 2**62),
                                              min(recent, 2**62), page_table.data_ptr(), lens.data_ptr(), keep.data_ptr(),
                                              0 if settled is None else settled.data_ptr(), 0 if evicted is None else evicted.data_ptr(), slots_at,
                                              *kp, *vp, weights.data_ptr(), w0, *((0,) if plain else ()), *w1[:-1], positions.data_ptr(), p0,
                                              *((0,) if plain else ()), *p1[:-1], places, rows, ws.data_ptr(), nbytes), _raw_stream(dev)), "kdn_evict")
