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

Two ways keep a stream's pages from growing with its whole past.  Where every anchor layer has a window, `anchor_slide` frees the
pages between the sinks and the window.  With `anchor_queries` (the anchor layers' query heads) the pool holds the weight that
each cached key got (`anchor_weights`, which the layers' steps add to), and `anchor_evict` cuts streams to the keys of largest
weight, of each layer and head its own.  A stream's tokens keep the positions that they had; `anchor_tokens` counts the places.
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence

import torch

from kdn import anchor, bounded, ops


class AnchorPlan:
    """One step of some streams over their pages (device tensors): rows of the new tokens in the pages, their positions,
    cu_seqlens of the new tokens, page_table and context_lens of the tokens before them, and the host's max_new and
    max_context.  keep: whether the new tokens have places (drafts that may be refused have none).  slots: each stream's row of
    the pool's weights, if it keeps any, and run: the most new tokens that add to them over the pages; in_order: whether no stream
    was cut by weight, which fills places out of order."""

    def __init__(self, keep, rows, positions, cu_seqlens, page_table, context_lens, max_new, max_context, all_rows=None, cu_all=None, slots=None,
                 run=64, in_order=True):
        self.keep, self.rows, self.positions, self.cu_seqlens = keep, rows, positions, cu_seqlens
        self.page_table, self.context_lens, self.max_new, self.max_context = page_table, context_lens, max_new, max_context
        self.all_rows, self.cu_all = all_rows, cu_all
        self.slots, self.run, self.in_order = slots, run, in_order


class HybridMemoryPool:
    def __init__(self, max_streams: int, max_seq_len: int, num_layers: int = 20, num_heads: int = 16,
                 val_dim: int = 64, lifted_dim: int = 512, device="cuda:0", anchor_layers: int = 0,
                 anchor_heads: int = 4, anchor_dim: int = 64, anchor_pages: Optional[int] = None, page_tokens: int = 16,
                 anchor_dtype: torch.dtype = torch.bfloat16, anchor_queries: Optional[int] = None):
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
            # of a stream: tokens that have no place any more; places whose positions are held; the fewest places to which it can go back
            self._gone, self._settled, self._least = {}, {}, {}
            self._weights = None
            if anchor_queries is not None:
                if anchor_queries < 1 or anchor_queries % anchor_heads:
                    raise ValueError(f"HybridMemoryPool: anchor_queries is a multiple of anchor_heads, got {anchor_queries} and {anchor_heads}")
                shape = (max_streams, anchor_layers, anchor_heads, -(-max_seq_len // page_tokens) * page_tokens)
                with torch.inference_mode(False):  # torch writes them too: wherever the pool is made, they can be written everywhere
                    self._weights = torch.zeros(shape, dtype=torch.float32, device=device)
                    self._positions = torch.zeros(shape, dtype=torch.int32, device=device)
                self._run = min(64, 32 // (anchor_queries // anchor_heads))

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
                self._gone[slot] = self._settled[slot] = self._least[slot] = 0
                if self._weights is not None:
                    self._weights[slot] = 0  # as those of all places behind a stream's last, until a step adds to them
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
                for t in (self._gone, self._settled, self._least):
                    t[child] = t[parent_stream_id]
                if self._weights is not None:
                    for t in (self._weights, self._positions):
                        t[child] = t[parent_stream_id]
        return child

    def release_stream(self, stream_id: int) -> None:
        try:
            self._pool.release(stream_id)
        except RuntimeError:
            return
        self.prompt_len.pop(stream_id, None)
        if self._anchor is not None:
            self._anchor.close(self._anchor_stream.pop(stream_id))
            del self._gone[stream_id], self._settled[stream_id], self._least[stream_id]

    # ---- the anchor layers' pages

    def anchor_pages(self, layer: int):
        """(k_pages, v_pages) of one anchor layer, (pages, heads, page_tokens, d) views of the slab."""
        return self.anchor_slab[:, layer, 0], self.anchor_slab[:, layer, 1]

    def _copy_pages(self, moves) -> None:
        # a host slab (bookkeeping alone) has nothing to copy, as the recurrent slab's forks
        if len(moves) and self.anchor_slab.is_cuda:
            anchor.page_copy(self.anchor_slab, moves)

    def anchor_weights(self, layer: int) -> torch.Tensor:
        """The weights of one anchor layer's keys, (max_streams, heads, places): what its steps are given."""
        if self._weights is None:
            raise ValueError("HybridMemoryPool: weights need anchor_queries")
        return self._weights[:, layer]

    def anchor_tokens(self, stream_id: int) -> int:
        """Places that the stream has in the pages."""
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
        first = [c + self._gone[s] for c, s in zip(context, streams)]  # the new tokens' positions start here
        keep = depths is None
        if not keep:
            depths = torch.as_tensor(depths)
            whole = not (depths.is_floating_point() or depths.is_complex() or depths.dtype is torch.bool)
            if depths.is_cuda or depths.shape != (sum(new_tokens),) or (depths.numel() and not whole):
                raise ValueError(f"anchor_plan: depths are {sum(new_tokens)} host integers, one a token; got {tuple(depths.shape)} {depths.dtype} "
                                 f"on {depths.device}")
            depths = depths.to(torch.int64)
        if keep:
            if self._weights is not None and max((c + n for c, n in zip(context, new_tokens)), default=0) > self._weights.shape[-1]:
                raise RuntimeError(f"anchor_plan: weights are held of {self._weights.shape[-1]} places a stream")
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
            parts += [torch.cat([torch.arange(c, c + n) for c, n in zip(first, new_tokens)] or [torch.empty(0, dtype=torch.int64)]),
                      torch.cat([self._anchor.rows(i, c, n) for i, c, n in zip(ids, context, new_tokens)] or [torch.empty(0, dtype=torch.int64)])]
        else:
            per = torch.repeat_interleave(torch.tensor(first, dtype=torch.int64), torch.tensor(new_tokens, dtype=torch.int64))
            parts += [per + depths]
        run = 64 if self._weights is None else self._run
        gather = keep and most > run and longest > 0  # a prompt's next piece reads its earlier keys whole
        if gather:
            parts += [torch.cat([self._anchor.rows(i, 0, c + n) for i, c, n in zip(ids, context, new_tokens)]),
                      torch.tensor([0, *(c + n for c, n in zip(context, new_tokens))]).cumsum(0)]
        if self._weights is not None:
            parts += [torch.tensor(list(streams), dtype=torch.int64)]
        flat = torch.cat([p.to(torch.int64) for p in parts])
        if dev.type == "cuda":
            flat = flat.pin_memory().to(dev, non_blocking=True)  # the allocator keeps the pinned copy until it is read
        out = list(flat.split([p.numel() for p in parts]))
        return AnchorPlan(keep, out[4] if keep else None, out[3], out[0], out[1].to(torch.int32).view(table.shape), out[2].to(torch.int32), most,
                          longest, *(out[-3 if self._weights is not None else -2:][:2] if gather else (None, None)),
                          slots=None if self._weights is None else out[-1].to(torch.int32), run=run,
                          in_order=not any(self._settled[s] for s in streams))

    def anchor_truncate(self, stream_id: int, tokens: int) -> None:
        """The stream's first `tokens` places stay; pages behind them are free.  Not back into places that an eviction filled out
        of order, nor to where a window reaches pages that have been freed; with 0 the stream begins anew."""
        if 0 < tokens < self._least[stream_id]:
            raise ValueError(f"anchor_truncate: stream {stream_id} goes back to {self._least[stream_id]} places at the least (an eviction filled those "
                             "before, or a window's pages are freed), or to none")
        had = self._anchor.length(self._anchor_stream[stream_id])
        self._anchor.truncate(self._anchor_stream[stream_id], tokens)
        if tokens == 0:
            self._gone[stream_id] = self._settled[stream_id] = self._least[stream_id] = 0
        if self._weights is not None and tokens < had:
            self._weights[stream_id, :, :, tokens:had] = 0  # (those behind a stream's last place are 0)

    def anchor_slide(self, streams: Sequence[int], window: int, sinks: int = 0) -> int:
        """Frees the pages that no token from now on sees in layers that all have this window and sinks (or smaller ones): those
        wholly between the sinks and the last window - 1 tokens; their number.  Plans made before are void."""
        window, sinks = anchor._window(window, sinks, "anchor_slide")
        if window == 0 or self._weights is not None:
            raise ValueError("anchor_slide: needs a window, and a pool that keeps no weights of the places")
        P, freed = self._anchor.page_tokens, 0
        for s in streams:
            i = self._anchor_stream[s]
            first, end = -(-sinks // P), max(self._anchor.length(i) - window + 1, 0) // P
            if end > first:
                self._anchor.drop(i, first, end - first)
                self._gone[s] += (end - first) * P
                self._least[s] = max(self._least[s], first * P + window - 1)
                freed += end - first
        return freed

    def anchor_evict(self, streams: Sequence[int], keep: int, sinks: int = 0, recent: int = 0) -> None:
        """Cuts each of the streams to `keep` places, in every layer and head to the positions below `sinks`, the last `recent` and,
        of the others, the keys of largest weight.  Where those are more than `keep`, the sinks and the latest keep - sinks stay.  If the pages
        do not suffice (a stream whose pages others share gets its own), RuntimeError, and no stream is cut.  Plans made before are
        void."""
        if self._weights is None:
            raise ValueError("HybridMemoryPool: weights need anchor_queries")
        keep = operator.index(keep)
        if keep < 0 or operator.index(sinks) < 0 or operator.index(recent) < 0:
            raise ValueError(f"anchor_evict: keep, sinks and recent are 0 or more, got {keep}, {sinks}, {recent}")
        recent = min(recent, max(keep - sinks, 0))  # of more than there is room for the lowest places would stay, the oldest tokens
        if len(set(streams)) != len(streams):
            raise ValueError("anchor_evict: a stream twice")
        long = [s for s in streams if self._anchor.length(self._anchor_stream[s]) > keep]
        if not long:
            return
        ids = [self._anchor_stream[s] for s in long]
        moves = []
        try:
            for i in ids:
                moves.append(self._anchor.own(i, keep))
        finally:  # copies that were granted are made, so that what the tables name is there
            self._copy_pages(torch.cat(moves) if moves else [])
        lens = [self._anchor.length(i) for i in ids]
        table = self._anchor.table(ids)
        parts = [table.flatten(), *(torch.tensor(x, dtype=torch.int32) for x in
                                    (lens, [keep] * len(ids), [self._settled[s] for s in long], [self._gone[s] for s in long], long))]
        dev = self.anchor_slab.device
        if dev.type == "cuda":
            flat = torch.cat(parts).pin_memory().to(dev, non_blocking=True)
            tab, *rest = flat.split([p.numel() for p in parts])
            n, k, settled, gone, slots = rest
            bounded.evict(self.anchor_slab[:, :, 0], self.anchor_slab[:, :, 1], tab.view(table.shape), n, k, self._weights, self._positions, settled,
                          gone, sinks=sinks, recent=recent, slots=slots, max_len=max(lens))
            self._weights[..., keep:max(lens)].index_fill_(0, slots.long(), 0)
        for s, i, L in zip(long, ids, lens):
            self._anchor.truncate(i, keep)
            self._gone[s] += L - keep
            self._settled[s] = self._least[s] = keep

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
