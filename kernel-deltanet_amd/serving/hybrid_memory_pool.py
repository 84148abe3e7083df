"""HybridMemoryPool -- the reference's slab pool API (serving/hybrid_memory_pool.h:40-85) over the native
slot bookkeeping of libkdn.so (kdn_pool_*) and one device slab of fp32 recurrent states.

Each stream owns one slot of [num_layers][num_heads][lifted_dim][val_dim] fp32 state (the layout the
decode and scan kernels read with unit stride); the pool allocates nothing after construction
(allocate / fork / release only move slots between the free stack and the active set; fork copies the
parent's slot on the device).

With `anchor_layers` the pool also holds the pages of the softmax anchor layers' keys and values (the reference's
16-token reference-counted pages, serving/hybrid_memory_pool.cpp:20-22, 62-84), in one slab
[anchor_pages][anchor_layers][2][anchor_heads][page_tokens][anchor_dim]: a stream's pages hold its tokens of all
anchor layers, fork_stream shares them (a stream that writes into a shared, partly filled page gets a copy of it
first), release_stream frees those that no other stream has.  `anchor_plan` makes room for a step's new tokens and
gives what the layers' kernels take, the same for all layers; nothing waits for the device.
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence

import torch

from kdn import anchor, ops


class AnchorPlan:
    """One step of some streams over their pages (device tensors): rows of the new tokens in the pages, their positions,
    cu_seqlens of the new tokens, page_table and context_lens of the tokens before them, and the host's max_new and
    max_context.  keep: whether the new tokens have places (drafts that may be refused have none)."""

    def __init__(self, keep, rows, positions, cu_seqlens, page_table, context_lens, max_new, max_context, all_rows=None, cu_all=None):
        self.keep, self.rows, self.positions, self.cu_seqlens = keep, rows, positions, cu_seqlens
        self.page_table, self.context_lens, self.max_new, self.max_context = page_table, context_lens, max_new, max_context
        self.all_rows, self.cu_all = all_rows, cu_all


class HybridMemoryPool:
    def __init__(self, max_streams: int, max_seq_len: int, num_layers: int = 20, num_heads: int = 16,
                 val_dim: int = 64, lifted_dim: int = 512, device="cuda:0", anchor_layers: int = 0,
                 anchor_heads: int = 4, anchor_dim: int = 64, anchor_pages: Optional[int] = None, page_tokens: int = 16,
                 anchor_dtype: torch.dtype = torch.bfloat16):
        self.max_streams = max_streams
        self.max_seq_len = max_seq_len
        self.num_layers = num_layers
        self._pool = ops.StatePool(max_streams, num_layers, num_heads, lifted_dim, val_dim, device=device)
        self.recurrent_bytes_per_stream = self._pool.slot_bytes
        self.prompt_len = {}
        self.anchor_layers, self._anchor = anchor_layers, None
        if anchor_layers:
            # by default room for every stream at its longest
            pages = max_streams * -(-max_seq_len // page_tokens) if anchor_pages is None else anchor_pages
            self._anchor = anchor.PagePool(pages, page_tokens, max_streams)
            self.anchor_slab = torch.empty(pages, anchor_layers, 2, anchor_heads, page_tokens, anchor_dim, dtype=anchor_dtype, device=device)
            self._anchor_stream = {}

    @property
    def slab(self) -> torch.Tensor:
        """[max_streams, num_layers, num_heads, lifted_dim, val_dim] fp32."""
        return self._pool.slab

    def layer_states(self, layer: int) -> torch.Tensor:
        """[max_streams, num_heads, lifted_dim, val_dim] view: the states argument of a layer's step."""
        return self._pool.layer_states(layer)

    def allocate_stream(self, prompt_len: int) -> int:
        slot = self._pool.allocate()
        if slot >= 0:
            self.prompt_len[slot] = prompt_len
            if self._anchor is not None:
                self._anchor_stream[slot] = self._anchor.open()
        return slot

    def fork_stream(self, parent_stream_id: int) -> int:
        try:
            child = self._pool.fork(parent_stream_id)
        except RuntimeError:
            return -1
        if child >= 0:
            self.prompt_len[child] = self.prompt_len.get(parent_stream_id, 0)
            if self._anchor is not None:
                self._anchor_stream[child] = self._anchor.fork(self._anchor_stream[parent_stream_id])
        return child

    def release_stream(self, stream_id: int) -> None:
        try:
            self._pool.release(stream_id)
        except RuntimeError:
            return
        self.prompt_len.pop(stream_id, None)
        if self._anchor is not None:
            self._anchor.close(self._anchor_stream.pop(stream_id))

    # ---- the anchor layers' pages

    def anchor_pages(self, layer: int):
        """(k_pages, v_pages) of one anchor layer, (pages, heads, page_tokens, d) views of the slab."""
        return self.anchor_slab[:, layer, 0], self.anchor_slab[:, layer, 1]

    def _copy_pages(self, moves) -> None:
        # a host slab (bookkeeping alone) has nothing to copy, as the recurrent slab's forks
        if len(moves) and self.anchor_slab.is_cuda:
            anchor.page_copy(self.anchor_slab, moves)

    def anchor_tokens(self, stream_id: int) -> int:
        return self._anchor.length(self._anchor_stream[stream_id])

    def anchor_plan(self, streams: Sequence[int], new_tokens: Sequence[int], depths: Optional[torch.Tensor] = None) -> AnchorPlan:
        """The step of `new_tokens[i]` more tokens of streams[i]: room is made for them (pages that are shared and partly
        filled are copied first).  With `depths` (host integers, one a token) the tokens are drafts, at positions context +
        depth, and no room is made: they may be refused.  If the pages do not suffice, RuntimeError, and no stream has
        changed."""
        if len(new_tokens) != len(streams):
            raise ValueError(f"anchor_plan: {len(streams)} streams and {len(new_tokens)} numbers of new tokens")
        new_tokens = [operator.index(n) for n in new_tokens]
        if min(new_tokens, default=0) < 0:
            raise ValueError(f"anchor_plan: numbers of new tokens are not negative, got {new_tokens}")
        ids = [self._anchor_stream[s] for s in streams]
        if len(set(ids)) != len(ids):
            raise ValueError("anchor_plan: a stream twice in one step")
        dev, P = self.anchor_slab.device, self._anchor.page_tokens
        context = [self._anchor.length(i) for i in ids]
        keep = depths is None
        if not keep:
            depths = torch.as_tensor(depths)
            whole = not (depths.is_floating_point() or depths.is_complex() or depths.dtype is torch.bool)
            if depths.is_cuda or depths.shape != (sum(new_tokens),) or (depths.numel() and not whole):
                raise ValueError(f"anchor_plan: depths are {sum(new_tokens)} host integers, one a token; got {tuple(depths.shape)} {depths.dtype} "
                                 f"on {depths.device}")
            depths = depths.to(torch.int64)
        if keep:
            moves, done = [], []
            try:
                for i, n in zip(ids, new_tokens):
                    moves += self._anchor.extend(i, n)
                    done.append(i)
            except BaseException:
                # the streams extended so far give their room back; copies that their shared pages got are made, so that
                # what their tables name is there
                for i, c in zip(done, context):
                    self._anchor.truncate(i, c)
                self._copy_pages(moves)
                raise
            self._copy_pages(moves)
        table = self._anchor.table(ids)
        offsets = [0]
        for n in new_tokens:
            offsets.append(offsets[-1] + n)
        most, longest = max(new_tokens, default=0), max(context, default=0)
        parts = [torch.tensor(offsets, dtype=torch.int64), table.flatten(), torch.tensor(context, dtype=torch.int64)]
        if keep:
            parts += [torch.cat([torch.arange(c, c + n) for c, n in zip(context, new_tokens)] or [torch.empty(0, dtype=torch.int64)]),
                      torch.cat([self._anchor.rows(i, c, n) for i, c, n in zip(ids, context, new_tokens)] or [torch.empty(0, dtype=torch.int64)])]
        else:
            per = torch.repeat_interleave(torch.tensor(context, dtype=torch.int64), torch.tensor(new_tokens, dtype=torch.int64))
            parts += [per + depths]
        gather = keep and most > 64 and longest > 0  # a prompt's next piece reads its earlier keys whole
        if gather:
            parts += [torch.cat([self._anchor.rows(i, 0, c + n) for i, c, n in zip(ids, context, new_tokens)]),
                      torch.tensor([0, *(c + n for c, n in zip(context, new_tokens))]).cumsum(0)]
        flat = torch.cat([p.to(torch.int64) for p in parts])
        if dev.type == "cuda":
            flat = flat.pin_memory().to(dev, non_blocking=True)  # the allocator keeps the pinned copy until it is read
        out = list(flat.split([p.numel() for p in parts]))
        return AnchorPlan(keep, out[4] if keep else None, out[3], out[0], out[1].to(torch.int32).view(table.shape), out[2].to(torch.int32), most,
                          longest, *(out[5:7] if gather else ()))

    def anchor_truncate(self, stream_id: int, tokens: int) -> None:
        """The stream's first `tokens` tokens stay; pages behind them are free."""
        self._anchor.truncate(self._anchor_stream[stream_id], tokens)

    def anchor_compact(self) -> int:
        """Moves the pages in use to the front of the slab; the number of pages moved.  Plans made before are void."""
        moves = self._anchor.compact()
        self._copy_pages(moves)
        return moves.shape[0]

    @property
    def anchor_pages_used(self) -> int:
        return self._anchor.used

    @property
    def anchor_pages_free(self) -> int:
        return self._anchor.free

    def get_total_allocated_bytes(self) -> int:
        return self._pool.allocated_bytes()

    def get_free_bytes(self) -> int:
        return self._pool.free_bytes()

    def print_memory_profile(self) -> None:
        active = self._pool.active
        total = self.max_streams * self.recurrent_bytes_per_stream
        used = self.get_total_allocated_bytes()
        print("[HybridMemoryPool]")
        print(f"  Active streams: {active} / {self.max_streams}")
        if self._anchor is not None:
            print(f"  Anchor pages: {self._anchor.used} / {self._anchor.num_pages} of {self._anchor.page_tokens} tokens")
        print(f"  Recurrent slab: {used / 2**20:.1f} MB / {total / 2**20:.1f} MB ({100.0 * used / max(total, 1):.1f}%)")
