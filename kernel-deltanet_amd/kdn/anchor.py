"""Operators of the softmax anchor layers (include/kdn_anchor.h): the attention layers that a hybrid model keeps between
its recurrent ones, and the pages their keys and values live in.

    rotary            positions of q and k, with gradients
    attention         causal attention over packed prompts with grouped heads, whole or in a window, with gradients
    PagePool          which pages a stream's tokens lie on: fork, extend, truncate, own, drop, compact, free (host)
    page_copy         whole pages (forks about to write, compaction)
    page_append       new tokens' keys and values into their pages
    tree_attention    one new token a stream, a run of them, or a tree of drafts, over the pages, whole or in a window; and what
                      weight each key got

torch supplies device memory and the current HIP stream; every computation is a HIP kernel in libkdn.so.  The tensors are
gfx950 device tensors, (tokens, heads, d) with d = 64 or 128 in bfloat16 or float32, in any strides with contiguous heads
that start on 16 bytes (others are copied first).  Nothing here waits for the device.  The reference's anchor pages are
serving/hybrid_memory_pool.{h,cpp}.
"""
from __future__ import annotations

import ctypes
import functools
import math
import operator
import struct
from typing import List, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N
from .ops import _HERE, _tag, forward_only, require_device

_ref = ctypes.byref
_BF16, _F32 = torch.bfloat16, torch.float32
_FAR = (2**31 - 1) // 64     # bytes from a row to the next that the kernels' copies reach over
_ODD_BF16, _ODD_F32 = ~(2**23 - 8), ~(2**22 - 4)  # bits that strides within reach of 16-byte rows do not have
_raw_stream, _this_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice

# The argument structs of include/kdn_anchor.h as packed bytes, in C's own alignment: a decode step's calls are host-bound,
# and a ctypes structure filled field by field takes as long as the rest of a call.  The order is that of the mirrors in
# kdn/_native.py (tests/test_anchor_host.py holds them against each other).
_ATTN = struct.Struct("@qqqqqiifPP" + 4 * "Pqq" + "P" + "Pqq")
_ATTN_BWD = struct.Struct("@P" + 4 * "Pqq" + "PN")
_ROTARY = struct.Struct("@qqqiiiiifPP" + 4 * "Pqq")
_APPEND = struct.Struct("@qqiiqqP" + 2 * "Pqq" + 2 * "Pqqq")
_TREE = struct.Struct("@qqqqqqiifqqqqPPPP" + 3 * "Pqq" + 2 * "Pqqq" + "Pqq" + "PN")
_BOUND = struct.Struct("@qqPqqqqP")  # include/kdn_bounded.h


def _device(index: int):
    """The context of work on a device, as ops._on."""
    return _HERE if index == _this_device() else torch.cuda.device(index)


def _heads(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None):
    """(t, its address, token stride, head stride), t as the library reads it: (tokens, heads, d), contiguous heads, rows on
    16 bytes (copied if they are not)."""
    if not t.is_cuda:
        require_device(t, what)
    if t.dim() != 3:
        raise ValueError(f"{what}: expects (tokens, heads, d), got {tuple(t.shape)}")
    dt = t.dtype
    if like is not None and (dt is not like.dtype or t.get_device() != like.get_device() or t.shape[2] != like.shape[2]):
        raise ValueError(f"{what}: expects {like.dtype} with d = {like.shape[-1]} on {like.device}; got {dt}, "
                         f"{tuple(t.shape)} on {t.device}")
    a, b, c = t.stride()
    p = t.data_ptr()
    if c != 1 or p & 15 or (a | b) & (_ODD_BF16 if dt is _BF16 else _ODD_F32):
        n, h, d = t.shape
        a, b = _steps(t)
        if c != 1 or p & 15 or (a | b) & (7 if dt is _BF16 else 3) or a > _FAR // dt.itemsize:
            # strides of an output of this shape: contiguous() leaves those of single tokens and heads as they were
            t, a, b = t.clone(memory_format=torch.contiguous_format), h * d, d
            p = t.data_ptr()
    return t, p, a, b


def _steps(t: torch.Tensor):
    """The strides of all dimensions but the last; of one that has a single entry, which may be any number, 0."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:-1], t.stride()))


def _out(t: torch.Tensor, what: str, shape, like: torch.Tensor):
    """As _heads, of an output that the caller gave: it is written where it is, so that it has to be in place."""
    require_device(t, what)
    if t.shape != shape or t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{what}: expects {tuple(shape)} {like.dtype} on {like.device}; got {tuple(t.shape)} {t.dtype} on {t.device}")
    a, b = _steps(t)
    if t.stride(-1) != 1 or t.data_ptr() % 16 or (a | b) * t.element_size() % 16:
        raise ValueError(f"{what}: needs contiguous heads whose rows start on 16 bytes")
    torch.autograd.graph.increment_version(t)  # as torch's own writes: a backward that saved it refuses what it has become
    return t, t.data_ptr(), a, b


def _new(like: torch.Tensor, shape):
    t = like.new_empty(shape)
    return t, t.data_ptr(), shape[1] * shape[2], shape[2]


def _ints(t: torch.Tensor, what: str, dtype: torch.dtype, dev: int, n: Optional[int] = None) -> torch.Tensor:
    if t.dtype is dtype and t.dim() == 1 and t.get_device() == dev and (n is None or t.shape[0] == n) and t.is_contiguous():
        return t
    require_device(t, what)
    if t.get_device() != dev or t.dim() != 1 or (n is not None and t.shape[0] != n) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: expects {'' if n is None else n} integers on GPU {dev}; got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.to(dtype).contiguous()


def _groups(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, what: str) -> None:
    if k.shape != v.shape or k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: k and v have one shape, and q a multiple of their heads; got q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")


def _dual(tensors) -> bool:
    """Whether one of them carries a forward-mode tangent, which a kernel's output would lose."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _tracked(*tensors) -> bool:
    """Whether autograd follows a call on them, in either mode (a Function without a forward mode refuses it by itself)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 and _dual(tensors)


def _scale(scale: Optional[float], d: int, what: str) -> float:
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (s > 0.0 and math.isfinite(s)):
        raise ValueError(f"{what}: scale must be positive, got {scale}")
    return s


def _window(window: Optional[int], sinks: int, what: str) -> Tuple[int, int]:
    """(window, sinks) as the library takes them; (0, 0) without a window."""
    n, s = 0 if window is None else operator.index(window), operator.index(sinks)
    if s < 0 or (window is not None and n < 1):
        raise ValueError(f"{what}: a window is 1 or more and sinks are 0 or more; got {window}, {sinks}")
    return (min(n, 2**62), min(s, 2**62)) if n else (0, 0)


# ------------------------------------------------------------------------------------------------- rotary positions


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained_length: int = 4096, low_turns: float = 1.0, high_turns: float = 32.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq (rotary_dim / 2,) float64 radians a position, magnitude) for `rotary`:

    - "none":   base^(-2j / rotary_dim);
    - "linear": all of them divided by `factor` (positions squeezed into the trained length);
    - "base":   the base raised to base * factor^(rotary_dim / (rotary_dim - 2)), so that the slowest pair slows by `factor`;
    - "parts":  a pair that turns at least `high_turns` times over `trained_length` keeps its frequency, one that turns at
                most `low_turns` times is divided by `factor`, those between go over linearly; the magnitude is
                1 + 0.1 ln(factor).
    """
    if rotary_dim <= 0 or rotary_dim % 2 or base <= 0 or factor <= 0 or not high_turns > low_turns:
        raise ValueError(f"rotary_frequencies: rotary_dim {rotary_dim} must be even, base {base} and factor {factor} positive, "
                         f"high_turns over low_turns")
    at = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("rotary_frequencies: scaling 'base' needs rotary_dim > 2")
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -at, 1.0
    f = base ** -at
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "parts":
        keep = ((trained_length * f / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0 + 0.1 * math.log(factor)
    raise ValueError(f"rotary_frequencies: scaling is none, linear, base or parts, got {scaling!r}")


def _rotate(q, k, positions, inv_freq, interleaved, magnitude, inverse, in_place):
    if in_place:
        q, qp, q0, q1 = _out(q, "rotary q", q.shape, q)
    else:
        q, qp, q0, q1 = _heads(q, "rotary q")
    n, H, d = q.shape
    dev = q.get_device()
    KV, kp, k0, k1 = 0, 0, 0, 0
    if k is not None:
        k, kp, k0, k1 = _out(k, "rotary k", k.shape, q) if in_place else _heads(k, "rotary k", q)
        KV = k.shape[1]
        if k.shape[0] != n or k.shape[2] != d:
            raise ValueError(f"rotary: q and k have the same tokens and d; got {tuple(q.shape)}, {tuple(k.shape)}")
    pos = _ints(positions, "rotary positions", torch.int64, dev, n)
    if inv_freq.get_device() != dev or inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not 0 < 2 * inv_freq.shape[0] <= d:
        raise ValueError(f"rotary: inv_freq is (rotary_dim / 2,) float64 on {q.device} with rotary_dim <= {d}; got "
                         f"{tuple(inv_freq.shape)} {inv_freq.dtype} on {inv_freq.device}")
    f = inv_freq.contiguous()
    qo, qop, qo0, qo1 = (q, qp, q0, q1) if in_place else _new(q, (n, H, d))
    ko, kop, ko0, ko1 = (k, kp, k0, k1) if in_place or k is None else _new(k, (n, KV, d))
    with _device(dev):
        N.check(N.lib().kdn_rotary(_ROTARY.pack(n, H, KV, d, 2 * f.shape[0], _tag(q.dtype, "rotary"), interleaved, inverse, magnitude,
                                                pos.data_ptr(), f.data_ptr(), qp, q0, q1, kp, k0, k1, qop, qo0, qo1, kop, ko0, ko1),
                                   _raw_stream(dev)), "kdn_rotary")
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, magnitude, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (interleaved, magnitude, inverse)
        return _rotate(q, k, positions, inv_freq, interleaved, magnitude, inverse, False)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        interleaved, magnitude, inverse = ctx.how
        gq, gk = rotary(dq, dk, positions, inv_freq, interleaved, magnitude, not inverse)  # differentiable in dq and dk itself
        return gq, gk, None, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
           magnitude: float = 1.0, inverse: bool = False, in_place: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q (tokens, H, d) and k (tokens, H_kv, d; or None) with each head's first rotary_dim = 2 len(inv_freq) values turned by
    positions (tokens,) * inv_freq (float64, `rotary_frequencies`), in one launch: pairs (2j, 2j + 1) if interleaved, else
    (j, j + rotary_dim / 2); times `magnitude`; by the negative angle if inverse.  in_place writes q and k themselves.
    Differentiable (not in place)."""
    if _tracked(q, k):
        if in_place:
            raise ValueError("rotary: in_place has no gradient")
        return _Rotary.apply(q, k, positions, inv_freq, bool(interleaved), float(magnitude), bool(inverse))
    return _rotate(q, k, positions, inv_freq, bool(interleaved), float(magnitude), bool(inverse), in_place)


# ------------------------------------------------------------------------------------------------- prompt attention


def _attn_inputs(q, k, v, cu_q, cu_k):
    """q, k, v as _heads gives them and the offsets, checked."""
    qs = _heads(q, "attention q")
    ks, vs = _heads(k, "attention k", q), _heads(v, "attention v", q)
    _groups(q, k, v, "attention")
    dev = q.get_device()
    if cu_q.dim() != 1 or cu_q.shape[0] < 1 or (cu_k is not None and cu_k.shape != cu_q.shape):
        raise ValueError("attention: cu_seqlens are (sequences + 1,), the same number for queries and keys")
    if cu_k is None and k.shape[0] != q.shape[0]:
        raise ValueError(f"attention: {q.shape[0]} queries and {k.shape[0]} keys need cu_seqlens_k")
    return (qs, ks, vs, _ints(cu_q, "attention cu_seqlens", torch.int64, dev),
            None if cu_k is None else _ints(cu_k, "attention cu_seqlens_k", torch.int64, dev))


def _pack_attn(qs, ks, vs, cu_q, cu_k, scale, y, lse, low) -> bytes:
    n, H, d = qs[0].shape
    return _ATTN.pack(cu_q.shape[0] - 1, n, ks[0].shape[0], H, ks[0].shape[1], d, _tag(qs[0].dtype, "attention"), scale,
                      cu_q.data_ptr(), 0 if cu_k is None else cu_k.data_ptr(), *qs[1:], *ks[1:], *vs[1:], *y[1:],
                      0 if lse is None else lse.data_ptr(), *((0, 0, 0) if low is None else low[1:]))


def attention_forward(q, k, v, cu_seqlens, cu_seqlens_k=None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                      return_lse: bool = False, return_low: bool = False, window: Optional[int] = None, sinks: int = 0):
    """`attention` without autograd: y; or with return_lse (y, lse (H, tokens) float32); or with return_low too (y, lse, low),
    low what rounding took from y (None in float32), which makes the gradients' dy . y exact."""
    qs, ks, vs, cu_q, cu_k = _attn_inputs(q, k, v, cu_seqlens, cu_seqlens_k)
    near, first = _window(window, sinks, "attention")
    n, H, d = q.shape
    y = _new(q, (n, H, d)) if out is None else _out(out, "attention out", q.shape, q)
    lse = q.new_empty((H, n), dtype=_F32) if return_lse or return_low else None
    low = _new(q, (n, H, d)) if return_low and q.dtype is _BF16 else None
    args = _pack_attn(qs, ks, vs, cu_q, cu_k, _scale(scale, d, "attention"), y, lse, low)
    dev = q.get_device()
    with _device(dev):
        if near:
            N.check(N.lib().kdn_attn_window_fwd(args, near, first, _raw_stream(dev)), "kdn_attn_window_fwd")
        else:
            N.check(N.lib().kdn_attn_fwd(args, _raw_stream(dev)), "kdn_attn_fwd")
    return (y[0], lse, None if low is None else low[0]) if return_low else (y[0], lse) if return_lse else y[0]


@functools.lru_cache(maxsize=64)
def _bwd_bytes(nseq: int, nq: int, nk: int, H: int, KV: int, d: int, dtype: int, window: int, sinks: int) -> int:
    """kdn_attn_bwd_workspace_bytes (or a window's), which reads sizes only."""
    fwd = ctypes.c_char_p(_ATTN.pack(nseq, nq, nk, H, KV, d, dtype, 1.0, 1, 1, *(0,) * 16))
    args = _ATTN_BWD.pack(ctypes.cast(fwd, ctypes.c_void_p).value, *(0,) * 14)
    return N.lib().kdn_attn_window_bwd_workspace_bytes(args, window, sinks) if window else N.lib().kdn_attn_bwd_workspace_bytes(args)


def attention_backward(q, k, v, y, lse, dy, cu_seqlens, cu_seqlens_k=None, scale: Optional[float] = None,
                       low: Optional[torch.Tensor] = None, window: Optional[int] = None, sinks: int = 0):
    """(dq, dk, dv) of `attention_forward`'s y, lse and low (optional) for dL/dy, in the inputs' dtype, the same bits every
    time."""
    near, first = _window(window, sinks, "attention backward")
    qs, ks, vs, cu_q, cu_k = _attn_inputs(q, k, v, cu_seqlens, cu_seqlens_k)
    ys, dys = _heads(y, "attention y", q), _heads(dy, "attention dy", q)
    if y.shape != q.shape or dy.shape != q.shape or tuple(lse.shape) != (q.shape[1], q.shape[0]) or lse.dtype is not _F32 or \
            lse.device != q.device:
        raise ValueError(f"attention backward: y and dy have q's shape {tuple(q.shape)}, lse is (H, tokens) float32 on {q.device}")
    lse = lse.contiguous()
    lows = None
    if low is not None:
        lows = _heads(low, "attention low", q)
        if low.shape != q.shape:
            raise ValueError(f"attention backward: low has q's shape {tuple(q.shape)}")
    dq, dk, dv = _new(q, tuple(q.shape)), _new(k, tuple(k.shape)), _new(v, tuple(v.shape))
    fwd = ctypes.c_char_p(_pack_attn(qs, ks, vs, cu_q, cu_k, _scale(scale, q.shape[-1], "attention"), ys, lse, lows))
    at = ctypes.cast(fwd, ctypes.c_void_p).value
    dev = q.get_device()
    with _device(dev):
        nbytes = _bwd_bytes(cu_q.shape[0] - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], _tag(q.dtype, "attention"),
                            near, first)
        ws = q.new_empty(nbytes, dtype=torch.uint8)
        args = _ATTN_BWD.pack(at, *dys[1:], *dq[1:], *dk[1:], *dv[1:], ws.data_ptr(), nbytes)
        if near:
            N.check(N.lib().kdn_attn_window_bwd(args, near, first, _raw_stream(dev)), "kdn_attn_window_bwd")
        else:
            N.check(N.lib().kdn_attn_bwd(args, _raw_stream(dev)), "kdn_attn_bwd")
    return dq[0], dk[0], dv[0]


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, window, sinks):
        y, lse, low = attention_forward(q, k, v, cu_q, cu_k, scale, return_lse=True, return_low=True, window=window, sinks=sinks)
        ctx.save_for_backward(q, k, v, y, lse, cu_q, cu_k, low)
        ctx.how = (window, sinks)
        ctx.scale = scale
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        q, k, v, y, lse, cu_q, cu_k, low = ctx.saved_tensors
        return (*attention_backward(q, k, v, y, lse, dy, cu_q, cu_k, ctx.scale, low, *ctx.how), None, None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
              cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, window: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    """Causal softmax attention of packed sequences: q (tokens, H, d), k and v (tokens, H_kv, d), sequence b the rows
    cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (integers on the device; rows outside the offsets are padding: zeros).  Or a
    uniform batch q (B, T, H, d), k and v (B, T, H_kv, d) without cu_seqlens.  H is a multiple of H_kv, query head h uses
    key head h / (H / H_kv).  With cu_seqlens_k the keys have lengths of their own, and a sequence's last query sees its
    last key: query i the keys j <= p = i + len_k - len_q (none: its row is zero).  scale: 1 / sqrt(d).
    With `window` a query sees of these only the last `window`, j > p - window, and the first `sinks`, j < sinks.

    Differentiable in q, k and v, once; gradients come in their dtype, summed in fp32 in a fixed order.  `out`: where y goes
    (without autograd).  A step that is captured into a graph needs leaves of which no eager graph is left (torch runs a leaf's
    part of the backward on the stream that it was first used on)."""
    if q.dim() == 4:
        if cu_seqlens is not None or cu_seqlens_k is not None or k.dim() != 4 or v.dim() != 4 or k.shape[:2] != q.shape[:2]:
            raise ValueError("attention: (B, T, heads, d) tensors take no cu_seqlens and have one B and T")
        B, T = q.shape[:2]
        cu = torch.arange(0, (B + 1) * T, T, device=q.device) if T > 0 else torch.zeros(B + 1, dtype=torch.int64, device=q.device)
        flat = [t.reshape(B * T, *t.shape[2:]) for t in (q, k, v)]
        y = attention(*flat, cu, scale=scale, out=None if out is None else out.view(B * T, *out.shape[2:]), window=window, sinks=sinks)
        return y.view(q.shape)
    if cu_seqlens is None:
        raise ValueError("attention: packed (tokens, heads, d) tensors need cu_seqlens")
    if _tracked(q, k, v):
        if out is not None:
            raise ValueError("attention: out has no gradient")
        return _Attention.apply(q, k, v, cu_seqlens, cu_seqlens_k, scale, window, sinks)
    return attention_forward(q, k, v, cu_seqlens, cu_seqlens_k, scale, out, window=window, sinks=sinks)


# ------------------------------------------------------------------------------------------------- pages


def _pages(t: torch.Tensor, what: str, like: torch.Tensor):
    """(t, its address, page, head and token strides); a cache is used where it is, never copied."""
    require_device(t, what)
    if t.dim() != 4 or t.dtype is not like.dtype or t.get_device() != like.get_device() or t.shape[3] != like.shape[2]:
        raise ValueError(f"{what}: expects (pages, heads, page_tokens, {like.shape[-1]}) {like.dtype} on {like.device}; got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    a, b, c, e = t.stride()
    p = t.data_ptr()
    odd = 7 if t.dtype is _BF16 else 3
    if (a | b | c) & odd:
        a, b, c = _steps(t)
    if e != 1 or p & 15 or (a | b | c) & odd:
        raise ValueError(f"{what}: needs contiguous rows that start on 16 bytes (a cache is used where it is, never copied)")
    return t, p, a, b, c


def _pairs(pairs) -> torch.Tensor:
    """A page copy's list as the library reads it, (n, 2) int32 on the host."""
    p = pairs if isinstance(pairs, torch.Tensor) else torch.as_tensor(pairs)
    if p.is_cuda:
        raise ValueError("page_copy: pairs are host numbers")
    if p.dtype is torch.int32 and p.dim() == 2 and p.shape[1] == 2 and p.is_contiguous():
        return p
    if p.numel() and (p.is_floating_point() or p.dtype is torch.bool or p.dim() > 2 or (p.dim() == 2 and p.shape[1] != 2)):
        raise ValueError(f"page_copy: pairs are (n, 2) whole numbers, got {tuple(p.shape)} {p.dtype}")
    wide = p.reshape(-1, 2)
    p = wide.to(torch.int32).contiguous()
    if not torch.equal(p.to(wide.dtype), wide):
        raise ValueError("page_copy: a page number is past 32 bits")
    return p


def page_copy(slab: torch.Tensor, pairs) -> None:
    """Page pairs[i][0] of slab (pages, ...; contiguous) to page pairs[i][1], for host pairs (a CPU int32 tensor (n, 2) or
    pairs of numbers) as `PagePool` gives them: no page is the target of two pairs, or a target and a source."""
    if not slab.is_cuda:
        require_device(slab, "page_copy")
    if slab.dim() < 2 or not slab.is_contiguous():
        raise ValueError("page_copy: the slab must be contiguous, pages first")
    p = _pairs(pairs)
    n = p.shape[0]
    if n == 0:
        return
    dev = slab.get_device()
    pages = slab.shape[0]
    with _device(dev):
        N.check(N.lib().kdn_page_copy(slab.data_ptr(), pages, slab.nbytes // max(pages, 1), p.data_ptr(), n, _raw_stream(dev)),
                "kdn_page_copy")


def page_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, rows: torch.Tensor) -> None:
    """k and v (tokens, H_kv, d) into k_pages and v_pages (pages, H_kv, page_tokens, d): token i to place
    rows[i] % page_tokens of page rows[i] / page_tokens (`PagePool.rows`); one whose row is negative or past the pages is
    skipped.  Rows are distinct.  The pages have no gradient: k and v that need one are refused."""
    if _tracked(k, v):
        raise ValueError("page_append: the pages have no gradient; call it under torch.no_grad() or detach k and v")
    ks, vs = _heads(k, "page_append k"), _heads(v, "page_append v", k)
    kp, vp = _pages(k_pages, "page_append k_pages", k), _pages(v_pages, "page_append v_pages", k)
    n, KV, d = k.shape
    if v.shape != k.shape or k_pages.shape != v_pages.shape or k_pages.shape[1] != KV:
        raise ValueError(f"page_append: k, v {tuple(k.shape)}, {tuple(v.shape)} and pages {tuple(k_pages.shape)}, {tuple(v_pages.shape)} differ")
    dev = k.get_device()
    r = _ints(rows, "page_append rows", torch.int64, dev, n)
    with _device(dev):
        N.check(N.lib().kdn_page_append(_APPEND.pack(n, KV, d, _tag(k.dtype, "page_append"), k_pages.shape[2], k_pages.shape[0], r.data_ptr(),
                                                     *ks[1:], *vs[1:], *kp[1:], *vp[1:]), _raw_stream(dev)), "kdn_page_append")


class PagePool:
    """Which pages the tokens of each stream lie on (kdn_page_pool_*; host numbers only).  Forks share their parent's pages;
    the first write into a shared, partly filled page gives the writer a copy of it (`extend` names the copy to make)."""

    def __init__(self, num_pages: int, page_tokens: int = 16, max_streams: int = 1024):
        self.num_pages, self.page_tokens, self.max_streams = int(num_pages), int(page_tokens), int(max_streams)
        self._h = ctypes.c_void_p()
        N.check(N.lib().kdn_page_pool_create(self.num_pages, self.page_tokens, self.max_streams, _ref(self._h)), "kdn_page_pool_create")

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                N.lib().kdn_page_pool_destroy(h)
            except Exception:  # the interpreter ends, and its modules are gone
                pass
            self._h = None

    @staticmethod
    def _num(status: int, what: str) -> int:
        if status < 0:
            N.check(int(status), what)
        return int(status)

    def open(self) -> int:
        """A new empty stream's number."""
        return self._num(N.lib().kdn_page_pool_open(self._h), "kdn_page_pool_open")

    def fork(self, stream: int) -> int:
        return self._num(N.lib().kdn_page_pool_fork(self._h, stream), "kdn_page_pool_fork")

    def close(self, stream: int) -> None:
        self._num(N.lib().kdn_page_pool_close(self._h, stream), "kdn_page_pool_close")

    def extend(self, stream: int, tokens: int) -> List[Tuple[int, int]]:
        """Room for `tokens` more; the page copies to make (none or one) before anything is written."""
        pair = (ctypes.c_int32 * 2)()
        n = self._num(N.lib().kdn_page_pool_extend(self._h, stream, tokens, pair), "kdn_page_pool_extend")
        return [(pair[0], pair[1])] if n else []

    def truncate(self, stream: int, tokens: int) -> None:
        self._num(N.lib().kdn_page_pool_truncate(self._h, stream, tokens), "kdn_page_pool_truncate")

    def length(self, stream: int) -> int:
        return self._num(N.lib().kdn_page_pool_length(self._h, stream), "kdn_page_pool_length")

    def table(self, streams: Sequence[int]) -> torch.Tensor:
        """(streams, widest) int32 page numbers (CPU; a row's rest is 0)."""
        width = max([-(-self.length(s) // self.page_tokens) for s in streams], default=0)
        t = torch.zeros(len(streams), width, dtype=torch.int32)
        for row, s in zip(t, streams):
            self._num(N.lib().kdn_page_pool_table(self._h, s, row.data_ptr(), width), "kdn_page_pool_table")
        return t

    def rows(self, stream: int, first: int, n: int) -> torch.Tensor:
        """Where tokens first .. first + n - 1 lie (int64, CPU), for `page_append`."""
        r = torch.empty(n, dtype=torch.int64)
        self._num(N.lib().kdn_page_pool_rows(self._h, stream, first, n, r.data_ptr()), "kdn_page_pool_rows")
        return r

    def compact(self) -> torch.Tensor:
        """Moves the pages in use to the lowest numbers: the copies to make, (n, 2) int32, before anything else."""
        pairs = torch.empty(self.num_pages, 2, dtype=torch.int32)
        return pairs[:self._num(N.lib().kdn_page_pool_compact(self._h, pairs.data_ptr(), self.num_pages), "kdn_page_pool_compact")]

    def own(self, stream: int, tokens: int) -> torch.Tensor:
        """The pages of the stream's first `tokens` tokens become its own (`evict` writes them): the copies to make, (n, 2) int32,
        before anything is written."""
        pairs = torch.empty(-(-max(tokens, 0) // self.page_tokens), 2, dtype=torch.int32)
        return pairs[:self._num(N.lib().kdn_page_pool_own(self._h, stream, tokens, pairs.data_ptr(), pairs.shape[0]), "kdn_page_pool_own")]

    def drop(self, stream: int, first: int, pages: int) -> None:
        """Takes full pages out of the stream, from its page `first` on; the ones behind move up."""
        self._num(N.lib().kdn_page_pool_drop(self._h, stream, first, pages), "kdn_page_pool_drop")

    @property
    def used(self) -> int:
        return int(N.lib().kdn_page_pool_used(self._h))

    @property
    def free(self) -> int:
        return int(N.lib().kdn_page_pool_free(self._h))


# ------------------------------------------------------------------------------------------------- attention over pages


def _key_weights(weights: torch.Tensor, slots: Optional[torch.Tensor], streams: int, heads: Tuple[int, ...], like: torch.Tensor, what: str):
    """(slots, their address or 0) of weights that a call writes where they are, (slots, *heads, places) float32 on like's device."""
    if not weights.is_cuda:
        require_device(weights, f"{what} weights")
    if weights.dim() != 2 + len(heads) or weights.shape[1:-1] != heads or weights.dtype is not _F32 or weights.get_device() != like.get_device() or \
            (weights.shape[-1] > 1 and weights.stride(-1) != 1):
        raise ValueError(f"{what}: weights are (slots, {', '.join(map(str, heads))}, places) float32 on {like.device}, places next to one another; "
                         f"got {tuple(weights.shape)} {weights.dtype} on {weights.device}")
    if weights.requires_grad:
        raise ValueError(f"{what}: weights have no gradient")
    if 0 in weights.stride() and any(s == 0 and n > 1 for s, n in zip(weights.stride(), weights.shape)):
        raise ValueError(f"{what}: weights are written where they are, and these lie on one another (an expanded tensor)")
    if slots is None:
        if weights.shape[0] != streams:
            raise ValueError(f"{what}: weights of {weights.shape[0]} slots for {streams} streams need slots")
        return None, 0
    slots = _ints(slots, f"{what} slots", torch.int32, like.get_device(), streams)
    return slots, slots.data_ptr()


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   page_table: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                   parents: Optional[torch.Tensor] = None, scale: Optional[float] = None, max_context: Optional[int] = None,
                   max_new: Optional[int] = None, out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                   window: Optional[int] = None, sinks: int = 0, weights: Optional[torch.Tensor] = None,
                   slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens over their streams' pages and over themselves.

    q (tokens, H, d), k and v (tokens, H_kv, d): the new tokens, stream b's the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1
    (none given: one token a stream).  k_pages, v_pages (pages, H_kv, page_tokens, d) in any strides; page_table
    (streams, width) int32 and context_lens (streams,) on the device.  A new token sees its stream's whole context, itself,
    and along `parents` (tokens,) the new tokens before it: parents[i] is the number, within the stream's new tokens, of the
    one that token i hangs on, a lower one than its own, or -1 for the context (none given: a run, each on the one before).
    At most 64 new tokens a stream; max_new (64, or 1 without cu_seqlens) and max_context (what page_table holds) bound
    them from the host, so that nothing is read back; the closer, the smaller the launch.  Rows outside the offsets are
    padding: zeros, as are those of a stream past max_new.  `workspace`: uint8, at least `tree_workspace_bytes`, for a caller
    that allocates once.  Not differentiable: y raises on backward.

    With `window` a new token, at position context + its depth (how many new tokens it sees besides itself), sees only the last
    `window` positions, its own among them, and the first `sinks`.

    `weights` (slots, H_kv, places) float32: to the weight of each key of a stream's context is added the sum of its softmax weights
    over the stream's new tokens and the query heads of its head, and those of the new tokens' own places, behind the
    context, are set to theirs.  `slots` (streams,): which row is a stream's (none given: its number), no two the same; of those out of
    range nothing is written.  Runs of tokens alone (no parents), at most 32 rows of new tokens and query heads to a key head."""
    what = "tree_attention"
    tracked = _tracked(q, k, v, k_pages, v_pages)
    if tracked and forward_ad._current_level >= 0 and _dual((q, k, v, k_pages, v_pages)):
        raise NotImplementedError("tree_attention: has no forward-mode derivative")
    qs = _heads(q, "tree_attention q")
    ks, vs = _heads(k, "tree_attention k", q), _heads(v, "tree_attention v", q)
    _groups(q, k, v, what)
    kp, vp = _pages(k_pages, "tree_attention k_pages", q), _pages(v_pages, "tree_attention v_pages", q)
    n, H, d = q.shape
    KV, (pages, heads, P, _) = k.shape[1], k_pages.shape
    if k.shape[0] != n or v_pages.shape != k_pages.shape or heads != KV:
        raise ValueError(f"tree_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and pages {tuple(k_pages.shape)}, {tuple(v_pages.shape)} "
                         f"do not go together")
    dev = q.get_device()
    if page_table.get_device() != dev or page_table.dim() != 2 or page_table.dtype is not torch.int32 or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"tree_attention: page_table is (streams, width) int32 on {q.device}, got {tuple(page_table.shape)} "
                         f"{page_table.dtype} on {page_table.device}")
    B, width = page_table.shape
    lens = _ints(context_lens, "tree_attention context_lens", torch.int32, dev, B)
    if cu_seqlens is None:
        if n != B:
            raise ValueError(f"tree_attention: {n} new tokens of {B} streams need cu_seqlens")
        cu, most = torch.arange(B + 1, device=q.device), 1 if max_new is None else int(max_new)
    else:
        cu, most = _ints(cu_seqlens, "tree_attention cu_seqlens", torch.int64, dev, B + 1), 64 if max_new is None else int(max_new)
    par = None if parents is None else _ints(parents, "tree_attention parents", torch.int32, dev, n)
    room = width * P
    ctx = room if max_context is None else min(int(max_context), room)
    near, first = _window(window, sinks, what)
    bound = None
    if weights is not None:
        if par is not None:
            raise ValueError("tree_attention: weights are of runs of tokens, not of trees (a refused draft would count)")
        slots, slots_at = _key_weights(weights, slots, B, (KV,), q, what)
        s0, s1, _ = weights.stride()
        bound = _BOUND.pack(near, first, weights.data_ptr(), s0, s1, weights.shape[2], weights.shape[0], slots_at)
        torch.autograd.graph.increment_version(weights)
    elif near:
        bound = _BOUND.pack(near, first, 0, 0, 0, 0, 0, 0)
    y = _new(q, (n, H, d)) if out is None else _out(out, "tree_attention out", q.shape, q)
    sizes = (B, n, most, ctx, H, KV, d, _tag(q.dtype, what), _scale(scale, d, what), P, pages, width, page_table.stride(0))
    with _device(dev):
        if workspace is None:
            workspace = q.new_empty(_tree_bytes(_TREE.pack(*sizes, *_NO_TENSORS), bound), dtype=torch.uint8)
        elif workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError(f"tree_attention: the workspace is contiguous on {q.device}")
        args = _TREE.pack(*sizes, cu.data_ptr(), lens.data_ptr(), page_table.data_ptr(), 0 if par is None else par.data_ptr(), *qs[1:], *ks[1:],
                          *vs[1:], *kp[1:], *vp[1:], *y[1:], workspace.data_ptr(), workspace.nbytes)
        if bound is None:
            N.check(N.lib().kdn_tree_attn(args, _raw_stream(dev)), "kdn_tree_attn")
        else:
            N.check(N.lib().kdn_tree_attn_bounded(args, bound, _raw_stream(dev)), "kdn_tree_attn_bounded")
    return forward_only(what, (y[0],), (q, k, v, k_pages, v_pages))[0] if tracked else y[0]


_NO_TENSORS = (0,) * 26  # the tensor fields of kdn_tree_attn_args, where only sizes are read


def _tree_bytes(args: bytes, bound: Optional[bytes]) -> int:
    return N.lib().kdn_tree_attn_workspace_bytes(args) if bound is None else N.lib().kdn_tree_attn_bounded_workspace_bytes(args, bound)


def tree_workspace_bytes(streams: int, H: int, H_kv: int, d: int, dtype: torch.dtype, page_tokens: int, max_context: int,
                         max_new: int = 1, window: Optional[int] = None, sinks: int = 0, weights: bool = False) -> int:
    """Bytes of `tree_attention`'s workspace for up to these sizes (0: not supported), with this window, with or without weights."""
    near, first = _window(window, sinks, "tree_attention")
    # (an address that only says that there are weights; each stream has a slot)
    bound = _BOUND.pack(near, first, 4 if weights else 0, 0, 0, 0, streams, 0) if near or weights else None
    return int(_tree_bytes(_TREE.pack(streams, streams, max_new, max_context, H, H_kv, d, _tag(dtype, "tree_attention"), 1.0, page_tokens, 1,
                                      -(-max_context // page_tokens), 0, *_NO_TENSORS), bound))
