"""Operators of the softmax anchor layers (include/kdn_anchor.h): the attention layers that a hybrid model keeps between
its recurrent ones, and the pages their keys and values live in.

    rotary            positions of q and k, with gradients
    attention         causal attention over packed prompts with grouped heads, with gradients
    PagePool          which pages a stream's tokens lie on: fork, extend, truncate, compact, free (host)
    page_copy         whole pages (forks about to write, compaction)
    page_append       new tokens' keys and values into their pages
    tree_attention    one new token a stream, a run of them, or a tree of drafts, over the pages

torch supplies device memory and the current HIP stream; every computation is a HIP kernel in libkdn.so.  The tensors are
gfx950 device tensors, (tokens, heads, d) with d = 64 or 128 in bfloat16 or float32, in any strides with contiguous heads
that start on 16 bytes (others are copied first).  Nothing here waits for the device.  The reference's anchor pages are
serving/hybrid_memory_pool.{h,cpp}.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _native as N
from .ops import _on, _stream, _tag, require_device

_ref = ctypes.byref


def _heads(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """t as the library reads it: (tokens, heads, d), contiguous heads, rows on 16 bytes."""
    require_device(t, what)
    if t.dim() != 3:
        raise ValueError(f"{what}: expects (tokens, heads, d), got {tuple(t.shape)}")
    if like is not None and (t.device != like.device or t.dtype != like.dtype or t.shape[-1] != like.shape[-1]):
        raise ValueError(f"{what}: expects {like.dtype} with d = {like.shape[-1]} on {like.device}; got {t.dtype}, "
                         f"{tuple(t.shape)} on {t.device}")
    size = t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * size % 16 for s in t.stride()[:2]):
        t = t.contiguous()  # a view that starts off 16 bytes may be contiguous already
        t = t.clone() if t.data_ptr() % 16 else t
    return t


def _out(t: torch.Tensor, what: str, shape, like: torch.Tensor) -> torch.Tensor:
    """An output that the caller gave: it is written where it is, so that it has to be in place."""
    require_device(t, what)
    if tuple(t.shape) != tuple(shape) or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{what}: expects {tuple(shape)} {like.dtype} on {like.device}; got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * t.element_size() % 16 for s in t.stride()[:2]):
        raise ValueError(f"{what}: needs contiguous heads whose rows start on 16 bytes")
    return t


def _ints(t: torch.Tensor, what: str, dtype: torch.dtype, dev: torch.device, n: Optional[int] = None) -> torch.Tensor:
    require_device(t, what)
    if t.device != dev or t.dim() != 1 or (n is not None and t.shape[0] != n) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: expects {'' if n is None else n} integers on {dev}; got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.to(dtype).contiguous()


def _set(a: ctypes.Structure, name: str, t: torch.Tensor) -> None:
    setattr(a, name, t.data_ptr())
    field = getattr(a, name + "_stride")
    for i in range(len(field)):
        field[i] = t.stride(i)


def _groups(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, what: str) -> None:
    if k.shape != v.shape or k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: k and v have one shape, and q a multiple of their heads; got q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")


def _scale(scale: Optional[float], d: int, what: str) -> float:
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (s > 0.0 and math.isfinite(s)):
        raise ValueError(f"{what}: scale must be positive, got {scale}")
    return s


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
    what = "rotary"
    dev = q.device
    if in_place:
        q, k = _out(q, "rotary q", q.shape, q), None if k is None else _out(k, "rotary k", k.shape, q)
    else:
        q, k = _heads(q, "rotary q"), None if k is None else _heads(k, "rotary k", q)
    n = q.shape[0]
    if k is not None and k.shape[0] != n:
        raise ValueError(f"{what}: q and k have the same tokens; got {tuple(q.shape)}, {tuple(k.shape)}")
    pos = _ints(positions, "rotary positions", torch.int64, dev, n)
    if inv_freq.device != dev or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not 0 < 2 * inv_freq.shape[0] <= q.shape[-1]:
        raise ValueError(f"{what}: inv_freq is (rotary_dim / 2,) float64 on {dev} with rotary_dim <= {q.shape[-1]}; got "
                         f"{tuple(inv_freq.shape)} {inv_freq.dtype} on {inv_freq.device}")
    f = inv_freq.contiguous()
    qo = q if in_place else torch.empty(q.shape, dtype=q.dtype, device=dev)
    ko = k if in_place or k is None else torch.empty(k.shape, dtype=k.dtype, device=dev)
    a = N.RotaryArgs()
    a.tokens, a.H, a.H_kv, a.d = n, q.shape[1], 0 if k is None else k.shape[1], q.shape[2]
    a.rotary_dim, a.dtype = 2 * f.shape[0], _tag(q.dtype, what)
    a.interleaved, a.inverse, a.magnitude = int(bool(interleaved)), int(bool(inverse)), float(magnitude)
    a.positions, a.inv_freq = pos.data_ptr(), f.data_ptr()
    _set(a, "q", q)
    _set(a, "q_out", qo)
    if k is not None:
        _set(a, "k", k)
        _set(a, "k_out", ko)
    with _on(dev):
        N.check(N.lib().kdn_rotary(_ref(a), _stream(dev)), "kdn_rotary")
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
        gq, gk = _rotate(dq, dk, positions, inv_freq, interleaved, magnitude, not inverse, False)
        return gq, gk, None, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
           magnitude: float = 1.0, inverse: bool = False, in_place: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q (tokens, H, d) and k (tokens, H_kv, d; or None) with each head's first rotary_dim = 2 len(inv_freq) values turned by
    positions (tokens,) * inv_freq (float64, `rotary_frequencies`), in one launch: pairs (2j, 2j + 1) if interleaved, else
    (j, j + rotary_dim / 2); times `magnitude`; by the negative angle if inverse.  in_place writes q and k themselves.
    Differentiable (not in place)."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if in_place:
            raise ValueError("rotary: in_place has no gradient")
        return _Rotary.apply(q, k, positions, inv_freq, bool(interleaved), float(magnitude), bool(inverse))
    return _rotate(q, k, positions, inv_freq, interleaved, magnitude, inverse, in_place)


# ------------------------------------------------------------------------------------------------- prompt attention


def _attn_args(q, k, v, cu_q, cu_k, scale, y, lse, low=None) -> N.AttnArgs:
    a = N.AttnArgs()
    a.num_seqs, a.total_q, a.total_k = cu_q.shape[0] - 1, q.shape[0], k.shape[0]
    a.H, a.H_kv, a.d, a.dtype, a.scale = q.shape[1], k.shape[1], q.shape[2], _tag(q.dtype, "attention"), scale
    a.cu_q, a.cu_k = cu_q.data_ptr(), None if cu_k is None else cu_k.data_ptr()
    for name, t in (("q", q), ("k", k), ("v", v), ("y", y)):
        _set(a, name, t)
    a.lse = None if lse is None else lse.data_ptr()
    if low is not None:
        _set(a, "y_low", low)
    return a


def _attn_inputs(q, k, v, cu_q, cu_k):
    q = _heads(q, "attention q")
    k, v = _heads(k, "attention k", q), _heads(v, "attention v", q)
    _groups(q, k, v, "attention")
    dev = q.device
    if cu_q.shape[0] < 1 or (cu_k is not None and cu_k.shape != cu_q.shape):
        raise ValueError("attention: cu_seqlens are (sequences + 1,), the same number for queries and keys")
    if cu_k is None and k.shape[0] != q.shape[0]:
        raise ValueError(f"attention: {q.shape[0]} queries and {k.shape[0]} keys need cu_seqlens_k")
    return (q, k, v, _ints(cu_q, "attention cu_seqlens", torch.int64, dev),
            None if cu_k is None else _ints(cu_k, "attention cu_seqlens_k", torch.int64, dev))


def attention_forward(q, k, v, cu_seqlens, cu_seqlens_k=None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                      return_lse: bool = False, return_low: bool = False):
    """`attention` without autograd: y; or with return_lse (y, lse (H, tokens) float32); or with return_low too (y, lse, low),
    low what rounding took from y (None in float32), which makes the gradients' dy . y exact."""
    q, k, v, cu_q, cu_k = _attn_inputs(q, k, v, cu_seqlens, cu_seqlens_k)
    y = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else _out(out, "attention out", q.shape, q)
    lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device) if return_lse else None
    low = torch.empty(q.shape, dtype=q.dtype, device=q.device) if return_low and q.dtype is torch.bfloat16 else None
    a = _attn_args(q, k, v, cu_q, cu_k, _scale(scale, q.shape[-1], "attention"), y, lse, low)
    with _on(q.device):
        N.check(N.lib().kdn_attn_fwd(_ref(a), _stream(q.device)), "kdn_attn_fwd")
    return (y, lse, low) if return_low else (y, lse) if return_lse else y


def attention_backward(q, k, v, y, lse, dy, cu_seqlens, cu_seqlens_k=None, scale: Optional[float] = None,
                       low: Optional[torch.Tensor] = None):
    """(dq, dk, dv) of `attention_forward`'s y, lse and low (optional) for dL/dy, in the inputs' dtype, the same bits every
    time."""
    q, k, v, cu_q, cu_k = _attn_inputs(q, k, v, cu_seqlens, cu_seqlens_k)
    y, dy = _heads(y, "attention y", q), _heads(dy, "attention dy", q)
    if y.shape != q.shape or dy.shape != q.shape or tuple(lse.shape) != (q.shape[1], q.shape[0]) or lse.dtype != torch.float32 or \
            lse.device != q.device:
        raise ValueError(f"attention backward: y and dy have q's shape {tuple(q.shape)}, lse is (H, tokens) float32 on {q.device}")
    lse = lse.contiguous()
    if low is not None:
        low = _heads(low, "attention low", q)
        if low.shape != q.shape:
            raise ValueError(f"attention backward: low has q's shape {tuple(q.shape)}")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    f = _attn_args(q, k, v, cu_q, cu_k, _scale(scale, q.shape[-1], "attention"), y, lse, low)
    a = N.AttnBwdArgs()
    a.fwd = ctypes.addressof(f)
    for name, t in (("dy", dy), ("dq", dq), ("dk", dk), ("dv", dv)):
        _set(a, name, t)
    with _on(q.device):
        nbytes = N.lib().kdn_attn_bwd_workspace_bytes(_ref(a))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
        N.check(N.lib().kdn_attn_bwd(_ref(a), _stream(q.device)), "kdn_attn_bwd")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale):
        y, lse, low = attention_forward(q, k, v, cu_q, cu_k, scale, return_lse=True, return_low=True)
        ctx.save_for_backward(q, k, v, y, lse, cu_q, cu_k, low)
        ctx.scale = scale
        return y

    @staticmethod
    def backward(ctx, dy):
        q, k, v, y, lse, cu_q, cu_k, low = ctx.saved_tensors
        return (*attention_backward(q, k, v, y, lse, dy, cu_q, cu_k, ctx.scale, low), None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
              cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal softmax attention of packed sequences: q (tokens, H, d), k and v (tokens, H_kv, d), sequence b the rows
    cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (integers on the device; rows past the last offset are padding: zeros).  Or a
    uniform batch q (B, T, H, d), k and v (B, T, H_kv, d) without cu_seqlens.  H is a multiple of H_kv, query head h uses
    key head h / (H / H_kv).  With cu_seqlens_k the keys have lengths of their own, and a sequence's last query sees its
    last key: query i the keys j <= i + len_k - len_q (none: its row is zero).  scale: 1 / sqrt(d).

    Differentiable in q, k and v; gradients come in their dtype, summed in fp32 in a fixed order.  `out`: where y goes
    (without autograd)."""
    if q.dim() == 4:
        if cu_seqlens is not None or cu_seqlens_k is not None or k.dim() != 4 or v.dim() != 4 or k.shape[:2] != q.shape[:2]:
            raise ValueError("attention: (B, T, heads, d) tensors take no cu_seqlens and have one B and T")
        B, T = q.shape[:2]
        cu = torch.arange(0, (B + 1) * T, T, device=q.device) if T > 0 else torch.zeros(B + 1, dtype=torch.int64, device=q.device)
        flat = [t.reshape(B * T, *t.shape[2:]) for t in (q, k, v)]
        y = attention(*flat, cu, scale=scale, out=None if out is None else out.view(B * T, *out.shape[2:]))
        return y.view(q.shape)
    if cu_seqlens is None:
        raise ValueError("attention: packed (tokens, heads, d) tensors need cu_seqlens")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
        if out is not None:
            raise ValueError("attention: out has no gradient")
        return _Attention.apply(q, k, v, cu_seqlens, cu_seqlens_k, scale)
    return attention_forward(q, k, v, cu_seqlens, cu_seqlens_k, scale, out)


# ------------------------------------------------------------------------------------------------- pages


def _pages(t: torch.Tensor, what: str, like: torch.Tensor) -> torch.Tensor:
    require_device(t, what)
    if t.dim() != 4 or t.dtype != like.dtype or t.device != like.device or t.shape[-1] != like.shape[-1]:
        raise ValueError(f"{what}: expects (pages, heads, page_tokens, {like.shape[-1]}) {like.dtype} on {like.device}; got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * t.element_size() % 16 for s in t.stride()[:3]):
        raise ValueError(f"{what}: needs contiguous rows that start on 16 bytes (a cache is used where it is, never copied)")
    return t


def page_copy(slab: torch.Tensor, pairs) -> None:
    """Page pairs[i][0] of slab (pages, ...; contiguous) to page pairs[i][1], for host pairs (a CPU int32 tensor (n, 2) or
    pairs of numbers) as `PagePool` gives them: no page is the target of two pairs, or a target and a source."""
    require_device(slab, "page_copy")
    if not slab.is_contiguous() or slab.dim() < 2:
        raise ValueError("page_copy: the slab must be contiguous, pages first")
    p = torch.as_tensor(pairs, dtype=torch.int32).reshape(-1, 2).contiguous()
    if p.is_cuda:
        raise ValueError("page_copy: pairs are host numbers")
    if p.shape[0] == 0:
        return
    nbytes = slab[0].numel() * slab.element_size()
    with _on(slab.device):
        N.check(N.lib().kdn_page_copy(slab.data_ptr(), slab.shape[0], nbytes, p.data_ptr(), p.shape[0], _stream(slab.device)),
                "kdn_page_copy")


def page_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, rows: torch.Tensor) -> None:
    """k and v (tokens, H_kv, d) into k_pages and v_pages (pages, H_kv, page_tokens, d): token i to place
    rows[i] % page_tokens of page rows[i] / page_tokens (`PagePool.rows`); one whose row is negative or past the pages is
    skipped.  Rows are distinct."""
    k = _heads(k, "page_append k")
    v = _heads(v, "page_append v", k)
    kp, vp = _pages(k_pages, "page_append k_pages", k), _pages(v_pages, "page_append v_pages", k)
    if k.shape != v.shape or kp.shape != vp.shape or kp.shape[1] != k.shape[1]:
        raise ValueError(f"page_append: k, v {tuple(k.shape)}, {tuple(v.shape)} and pages {tuple(kp.shape)}, {tuple(vp.shape)} differ")
    r = _ints(rows, "page_append rows", torch.int64, k.device, k.shape[0])
    a = N.PageAppendArgs()
    a.tokens, a.H_kv, a.d, a.dtype = k.shape[0], k.shape[1], k.shape[2], _tag(k.dtype, "page_append")
    a.page_tokens, a.num_pages, a.rows = kp.shape[2], kp.shape[0], r.data_ptr()
    for name, t in (("k", k), ("v", v), ("k_pages", kp), ("v_pages", vp)):
        _set(a, name, t)
    with _on(k.device):
        N.check(N.lib().kdn_page_append(_ref(a), _stream(k.device)), "kdn_page_append")


class PagePool:
    """Which pages the tokens of each stream lie on (kdn_page_pool_*; host numbers only).  Forks share their parent's pages;
    the first write into a shared, partly filled page gives the writer a copy of it (`extend` names the copy to make)."""

    def __init__(self, num_pages: int, page_tokens: int = 16, max_streams: int = 1024):
        self.num_pages, self.page_tokens, self.max_streams = int(num_pages), int(page_tokens), int(max_streams)
        self._h = ctypes.c_void_p()
        N.check(N.lib().kdn_page_pool_create(self.num_pages, self.page_tokens, self.max_streams, _ref(self._h)), "kdn_page_pool_create")

    def __del__(self):
        if getattr(self, "_h", None):
            N.lib().kdn_page_pool_destroy(self._h)
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

    @property
    def used(self) -> int:
        return int(N.lib().kdn_page_pool_used(self._h))

    @property
    def free(self) -> int:
        return int(N.lib().kdn_page_pool_free(self._h))


# ------------------------------------------------------------------------------------------------- attention over pages


def _tree_args(q, k, v, k_pages, v_pages, page_table, num_seqs, max_context, max_new, scale) -> N.TreeAttnArgs:
    a = N.TreeAttnArgs()
    a.num_seqs, a.total_new, a.max_new, a.max_context = num_seqs, q.shape[0], max_new, max_context
    a.H, a.H_kv, a.d, a.dtype, a.scale = q.shape[1], k.shape[1], q.shape[2], _tag(q.dtype, "tree_attention"), scale
    a.page_tokens, a.num_pages = k_pages.shape[2], k_pages.shape[0]
    a.table_width, a.table_stride = page_table.shape[1], page_table.stride(0)
    return a


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   page_table: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                   parents: Optional[torch.Tensor] = None, scale: Optional[float] = None, max_context: Optional[int] = None,
                   max_new: Optional[int] = None, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens over their streams' pages and over themselves.

    q (tokens, H, d), k and v (tokens, H_kv, d): the new tokens, stream b's the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1
    (none given: one token a stream).  k_pages, v_pages (pages, H_kv, page_tokens, d) in any strides; page_table
    (streams, width) int32 and context_lens (streams,) on the device.  A new token sees its stream's whole context, itself,
    and along `parents` (tokens,) the new tokens before it: parents[i] is the number, within the stream's new tokens, of the
    one that token i hangs on, a lower one than its own, or -1 for the context (none given: a run, each on the one before).
    At most 64 new tokens a stream; max_new (64, or 1 without cu_seqlens) and max_context (what page_table holds) bound
    them from the host, so that nothing is read back; the closer, the smaller the launch.  `workspace`: uint8, at least
    `tree_workspace_bytes`, for a caller that allocates once."""
    q = _heads(q, "tree_attention q")
    k, v = _heads(k, "tree_attention k", q), _heads(v, "tree_attention v", q)
    _groups(q, k, v, "tree_attention")
    dev = q.device
    kp, vp = _pages(k_pages, "tree_attention k_pages", q), _pages(v_pages, "tree_attention v_pages", q)
    if k.shape[0] != q.shape[0] or kp.shape != vp.shape or kp.shape[1] != k.shape[1]:
        raise ValueError(f"tree_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and pages {tuple(kp.shape)}, {tuple(vp.shape)} do not go together")
    require_device(page_table, "tree_attention page_table")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != dev or (page_table.shape[1] and page_table.stride(1) != 1):
        raise ValueError(f"tree_attention: page_table is (streams, width) int32 on {dev}, got {tuple(page_table.shape)} {page_table.dtype}")
    B = page_table.shape[0]
    lens = _ints(context_lens, "tree_attention context_lens", torch.int32, dev, B)
    if cu_seqlens is None:
        if q.shape[0] != B:
            raise ValueError(f"tree_attention: {q.shape[0]} new tokens of {B} streams need cu_seqlens")
        cu, most = torch.arange(B + 1, device=dev), 1 if max_new is None else int(max_new)
    else:
        cu, most = _ints(cu_seqlens, "tree_attention cu_seqlens", torch.int64, dev, B + 1), 64 if max_new is None else int(max_new)
    par = None if parents is None else _ints(parents, "tree_attention parents", torch.int32, dev, q.shape[0])
    room = page_table.shape[1] * kp.shape[2]
    most_context = room if max_context is None else min(int(max_context), room)
    y = torch.empty(q.shape, dtype=q.dtype, device=dev) if out is None else _out(out, "tree_attention out", q.shape, q)
    a = _tree_args(q, k, v, kp, vp, page_table, B, most_context, most, _scale(scale, q.shape[-1], "tree_attention"))
    a.cu_new, a.context_lens, a.page_table = cu.data_ptr(), lens.data_ptr(), page_table.data_ptr()
    a.parents = None if par is None else par.data_ptr()
    for name, t in (("q", q), ("k", k), ("v", v), ("k_pages", kp), ("v_pages", vp), ("y", y)):
        _set(a, name, t)
    with _on(dev):
        ws = workspace
        if ws is None:
            ws = torch.empty(N.lib().kdn_tree_attn_workspace_bytes(_ref(a)), dtype=torch.uint8, device=dev)
        elif ws.device != dev or not ws.is_contiguous():
            raise ValueError(f"tree_attention: the workspace is contiguous on {dev}")
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
        N.check(N.lib().kdn_tree_attn(_ref(a), _stream(dev)), "kdn_tree_attn")
    return y


def tree_workspace_bytes(streams: int, H: int, H_kv: int, d: int, dtype: torch.dtype, page_tokens: int, max_context: int,
                         max_new: int = 1) -> int:
    """Bytes of `tree_attention`'s workspace for up to these sizes (0: not supported)."""
    a = N.TreeAttnArgs()
    a.num_seqs, a.total_new, a.max_new, a.max_context = streams, streams, max_new, max_context
    a.H, a.H_kv, a.d, a.dtype, a.scale = H, H_kv, d, _tag(dtype, "tree_attention"), 1.0
    a.page_tokens, a.num_pages, a.table_width = page_tokens, 1, -(-max_context // page_tokens)
    return int(N.lib().kdn_tree_attn_workspace_bytes(_ref(a)))
