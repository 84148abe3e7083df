"""Softmax anchor layer: the attention layer that a hybrid model keeps between its Kernel-DeltaNet layers, on the operators
of kdn.anchor.

    AnchorAttentionLayer(d_model, num_heads, num_kv_heads=None, rotary_dim=None, ...)
    .forward(x, cu_seqlens=None)       training and whole prompts: rotary positions, packed causal attention, projections;
                                       x (B, T, d_model), or packed (tokens, d_model) with cu_seqlens
    .step(x, plan, k_pages, v_pages)   serving: new tokens of streams whose keys and values live in pages
                                       (HybridMemoryPool.anchor_plan); one token a stream, a run of them, or a tree of drafts

A layer with a `window` sees the last `window` positions and the first `sinks` alone (HybridMemoryPool.anchor_slide frees the pages
between).  A step that is given the pool's weights (HybridMemoryPool.anchor_weights) adds to them what each key gets, by which
HybridMemoryPool.anchor_evict chooses what stays.

The reference keeps pages for such layers (serving/hybrid_memory_pool.{h,cpp}) and leaves the layers to its host framework.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from kdn import anchor, bounded

_RUN = 64  # new tokens that tree_attention takes of a stream


class AnchorAttentionLayer(nn.Module):
    def __init__(self, d_model: int, num_heads: int, num_kv_heads: Optional[int] = None, d_head: Optional[int] = None,
                 rotary_dim: Optional[int] = None, interleaved: bool = False, base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, trained_length: int = 4096, window: Optional[int] = None, sinks: int = 0):
        super().__init__()
        anchor._window(window, sinks, "AnchorAttentionLayer")
        self.window, self.sinks = window, sinks
        self.num_heads, self.num_kv_heads = num_heads, num_heads if num_kv_heads is None else num_kv_heads
        self.d_head = d_model // num_heads if d_head is None else d_head
        if self.d_head not in (64, 128) or num_heads % self.num_kv_heads:
            raise ValueError(f"AnchorAttentionLayer: heads of 64 or 128, num_heads a multiple of num_kv_heads; got d_head = {self.d_head}, "
                             f"{num_heads} over {self.num_kv_heads}")
        self.interleaved = interleaved
        self.w_q = nn.Linear(d_model, num_heads * self.d_head, bias=False)
        self.w_k = nn.Linear(d_model, self.num_kv_heads * self.d_head, bias=False)
        self.w_v = nn.Linear(d_model, self.num_kv_heads * self.d_head, bias=False)
        self.w_out = nn.Linear(num_heads * self.d_head, d_model, bias=False)
        frequencies = dict(rotary_dim=self.d_head if rotary_dim is None else rotary_dim, base=base, scaling=scaling, factor=factor,
                           trained_length=trained_length)
        with torch.inference_mode(False):  # a table that training can save, wherever the layer is made
            self._host_freq, self.magnitude = anchor.rotary_frequencies(**frequencies, device="cpu")
        self._inv_freq = self._host_freq
        self._follow()

    def _place(self, device) -> None:
        """The frequencies on `device`: float64 whatever the module's type is cast to (so no buffer), and there when this
        returns, for any stream: a copy from pageable host memory is waited for."""
        with torch.inference_mode(False):
            self._inv_freq = self._host_freq.to(device)

    def _follow(self) -> None:
        device = next(self.parameters(), self._inv_freq).device  # (projections may be replaced by ones without parameters)
        if self._inv_freq.device != device:
            self._place(device)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._follow()
        return self

    def inv_freq(self, device) -> torch.Tensor:
        """The frequencies on `device`: they move with the module.  Where its parameters came there by another way (assigned,
        or a replica's), they are brought there now, which a graph's capture cannot do."""
        if self._inv_freq.device != device:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AnchorAttentionLayer: move the module to its device, or call it once, before a capture")
            self._place(device)
        return self._inv_freq

    def _project(self, x: torch.Tensor, positions: torch.Tensor):
        n = x.shape[0]
        q = self.w_q(x).view(n, self.num_heads, self.d_head)
        k = self.w_k(x).view(n, self.num_kv_heads, self.d_head)
        v = self.w_v(x).view(n, self.num_kv_heads, self.d_head)
        q, k = anchor.rotary(q, k, positions, self.inv_freq(x.device), self.interleaved, self.magnitude)
        return q, k, v

    def forward(self, x: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Differentiable.  With cu_seqlens (device, the first 0) positions start anew in each sequence."""
        if cu_seqlens is None:
            B, T, _ = x.shape
            flat, cu = x.reshape(B * T, x.shape[-1]), torch.arange(B + 1, device=x.device) * T
            at = torch.arange(T, device=x.device).repeat(B)
        else:
            flat, cu = x, cu_seqlens.to(torch.int64)
            t = torch.arange(x.shape[0], device=x.device)
            at = t - cu[(torch.bucketize(t, cu, right=True) - 1).clamp(min=0)]
        q, k, v = self._project(flat, at)
        y = anchor.attention(q, k, v, cu, window=self.window, sinks=self.sinks)
        return self.w_out(y.view(-1, self.num_heads * self.d_head)).view(x.shape)

    @torch.no_grad()
    def step(self, x: torch.Tensor, plan, k_pages: torch.Tensor, v_pages: torch.Tensor, parents: Optional[torch.Tensor] = None,
             weights: Optional[torch.Tensor] = None):
        """x (tokens, d_model), the new tokens of plan's streams, against this layer's pages.  Returns the layer's output; for
        a plan of drafts (`keep` false) (output, k, v), of which the caller puts the accepted ones into the pages
        (anchor.page_append at the rows of a plan made for them).  `weights`: this layer's, to be added to.  Drafts add nothing, since
        they may be refused: where a pool keeps weights, the accepted ones' rows of x go through step once more, as a run of the plan made for
        them, which puts them into the pages and adds what the cached keys got from them."""
        if self.window is not None and not plan.in_order:
            raise ValueError("AnchorAttentionLayer: a window has no meaning over places that an eviction has filled out of order")
        weights = weights if plan.keep else None
        if weights is not None and plan.slots is None:
            raise ValueError("AnchorAttentionLayer: the plan's pool keeps no weights")
        q, k, v = self._project(x, plan.positions)
        if plan.keep:
            anchor.page_append(k, v, k_pages, v_pages, plan.rows)
        how = dict(window=self.window, sinks=self.sinks)
        if plan.max_new <= (_RUN if weights is None else plan.run):
            y = anchor.tree_attention(q, k, v, k_pages, v_pages, plan.page_table, plan.context_lens, plan.cu_seqlens, parents,
                                      max_context=plan.max_context, max_new=plan.max_new, weights=weights,
                                      slots=None if weights is None else plan.slots, **how)
        elif parents is not None or not plan.keep:
            raise ValueError(f"AnchorAttentionLayer: at most {_RUN} drafts a stream, got {plan.max_new}")
        else:
            cu_all = None
            if plan.max_context > 0:  # a prompt's next piece: its stream's keys so far out of the pages
                page, off = plan.all_rows // k_pages.shape[2], plan.all_rows % k_pages.shape[2]
                k, v, cu_all = k_pages[page, :, off], v_pages[page, :, off], plan.cu_all
            if weights is None:
                y = anchor.attention(q, k, v, plan.cu_seqlens, cu_all, **how)
            else:
                y, lse = anchor.attention_forward(q, k, v, plan.cu_seqlens, cu_all, return_lse=True, **how)
                bounded.attention_weights(q, k, lse, weights, plan.cu_seqlens, cu_all, add=True, slots=plan.slots, **how)
        out = self.w_out(y.view(-1, self.num_heads * self.d_head))
        return out if plan.keep else (out, k, v)
