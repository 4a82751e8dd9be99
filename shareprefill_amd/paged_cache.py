"""A key / value cache in pages for serving: pools, block tables and a stack of unused pages, all on the GPU.

    cache = PagedKVCache(num_layers=32, num_pages=4096, num_kv_heads=8, head_dim=128, max_requests=16, max_tokens=131072)
    cache.begin_step(new_lens, max_new_tokens=512)          # tokens each request brings (0: none): prompts in chunks, next tokens
    for layer in range(32):                                 # q, k, v of the step's tokens, request after request
        cache.write(layer, k, v)
        out = cache.attend(layer, q, softmax_scale)
    cache.begin_step(active=running)                        # a token of each running request, rows request by request
    cache.release(finished)

Requests that share the start of their prompt are rows of a group (group_sizes): the first row caches it, share() gives its whole pages to the others, and
attend reads them once for the group.  With key_weights the cache knows what attention every key has received, from each next token (attend) and from a
prompt's last ones (observe), and evict() keeps the heaviest of a request's keys when it holds too many:

    cache = PagedKVCache(..., group_sizes=[16, 16], key_weights=True)
    cache.begin_step(prompt_lens, max_new_tokens=8192)      # the common start, to rows 0 and 16
    ...
    cache.share(0, 4000), cache.share(1, 2500)              # rows 1 .. 15 and 17 .. 31 begin behind it
    cache.evict(budget=2048, recent=128, sinks=4)

A step (begin_step, write, attend, observe) reads no device value on the host, so it can be recorded into a HIP graph and replayed with other lengths;
share, join, evict and release run between steps.  The reference keeps no cache of its own (its decode step reads a contiguous one, shareprefill_attn.py:146-155).
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import ops


class PagedKVCache:
    """Requests are rows 0 .. max_requests - 1 of the block table; one model runs its steps in order on one stream."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, max_requests: int, max_tokens: int,
                 page_size: int = 64, device="cuda", group_sizes: Optional[Sequence[int]] = None, key_weights: bool = False):
        """group_sizes: rows that share prompts' starts, group after group from row 0 on; rows behind them share nothing."""
        if min(num_layers, num_pages, num_kv_heads, head_dim, max_requests, max_tokens) < 1:
            raise ValueError("every size of a PagedKVCache must be at least 1")
        self.page_size, self.num_pages, self.max_requests = page_size, num_pages, max_requests
        self.pools = torch.zeros(num_layers, 2, num_pages, num_kv_heads, page_size, head_dim, dtype=torch.bfloat16, device=device)
        dev = self.pools.device
        self.block_table = torch.full((max_requests, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        # (one place more than there are pages: where release puts what is none)
        self._stack = torch.arange(num_pages, -1, -1, dtype=torch.int32, device=dev).roll(-1)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=dev)
        self._one_each = torch.ones(max_requests, dtype=torch.int32, device=dev)
        self.tables: Optional[ops.PageTables] = None
        self._cu_q: Optional[torch.Tensor] = None
        self._seen_lens: Optional[torch.Tensor] = None  # of a step: keys that a request's rows may see
        sizes = list(group_sizes or [])
        if any(n < 1 for n in sizes) or sum(sizes) > max_requests:
            raise ValueError(f"group_sizes {sizes} must be at least 1 each and {max_requests} in all at most")
        if (sizes or key_weights) and max_requests > 1024:
            raise ValueError(f"max_requests {max_requests}: with group_sizes or key_weights there are at most 1024")
        starts = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
        ints = lambda x, dtype: torch.tensor(x, dtype=dtype, device=dev)
        self._group_starts = starts
        self.cu_groups = ints(starts, torch.int32)
        self.shared_lens = torch.zeros(len(sizes), dtype=torch.int32, device=dev)
        group_of = [i for i, n in enumerate(sizes) for _ in range(n)]
        self._group_of = ints(group_of + [len(sizes)] * (max_requests - len(group_of)), torch.int64)  # (none: one past the last)
        # keys at the front of a request that lie in pages of several, and that its group shares as long as the first row is there
        self._held = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self._joined = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self._shared_dropped = torch.zeros(len(sizes) + 1, dtype=torch.int32, device=dev)
        self._in_place = torch.zeros(max_requests, dtype=torch.int32, device=dev)  # of what has dropped some: keys at its front in front of all of them
        self._holder = ints([starts[i] for i in group_of] + list(range(len(group_of), max_requests)), torch.int64)
        # what attention every key has received, by its place in the pages (None: not kept), and how many keys evictions have taken from a request
        self.weights = torch.zeros(num_layers, num_pages, num_kv_heads, page_size, dtype=torch.float32, device=dev) if key_weights else None
        self.dropped = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.lost = torch.zeros(max_requests, dtype=torch.bool, device=dev)  # requests whose keys an eviction has spoilt
        self._last = None  # of a step: rows of its requests' last tokens (observe)

    def _check_mask(self, mask: torch.Tensor, name: str) -> None:
        if mask.dtype is not torch.bool or tuple(mask.shape) != (self.max_requests,) or mask.device != self.lens.device:
            raise ValueError(f"{name} must be bool [{self.max_requests}] on {self.lens.device}")

    def begin_step(self, new_lens: Optional[torch.Tensor] = None, max_new_tokens: Optional[int] = None,
                   active: Optional[torch.Tensor] = None) -> ops.PageTables:
        """Makes room for new_lens[r] more tokens of every request (int32 [max_requests]).  Without new_lens it is one token of every request that
        has active[r] (bool [max_requests]), and row r of the step's q, k and v is request r's: rows of the others go nowhere, and come out of attend as
        zeros.  Without either it is one of each of the max_requests rows, also of those that no request has: for a full server.  (A prompt that
        comes to such a row later would stand behind what was cached there.)

        max_new_tokens: how many there can be in all, the T of the step's q, k and v; tokens past it, of the last requests, are left out (the
        result's cu_new says what each request brought, and its lens grow by that).  Whether the pages sufficed is in the result's free_left
        (negative: they did not; tokens without a slot are not cached and seen by nobody).  positions count what evictions have dropped: a token's
        place in its request, not in the cache."""
        singles = new_lens is None
        if active is not None:
            if not singles:
                raise ValueError("new_lens already says which requests bring tokens: active is for steps without it")
            self._check_mask(active, "active")
        if singles:
            new_lens, max_new_tokens = self._one_each if active is None else active.to(torch.int32), self.max_requests
        elif max_new_tokens is None:
            raise ValueError("max_new_tokens: how many new tokens there can be in all")
        t = ops.page_tables(self.lens, new_lens, self.block_table, self._stack[:self.num_pages], self.free_count, self.page_size,
                            self.num_pages, max_new_tokens, truncate=not singles)
        self.lens.copy_(t.seq_lens)
        torch.clamp(t.free_left, min=0, out=self.free_count)
        self._seen_lens = t.seq_lens
        if active is not None:
            # from a token's place among the step's, which only active requests have, to its request's row (row r has r places in front of it at most)
            place = t.cu_new[:-1]
            t = t._replace(slots=torch.where(active, t.slots.index_select(0, place), -1), positions=t.positions.index_select(0, place) * new_lens)
            self._seen_lens = t.seq_lens * new_lens
        if self.weights is not None:
            # (places without a token stay at 0)
            if singles:
                t = t._replace(positions=t.positions + self.dropped * new_lens)
            else:
                token = torch.arange(t.positions.numel(), dtype=torch.int32, device=self.lens.device)
                row = torch.searchsorted(t.cu_new[1:], token, right=True).clamp_(max=self.max_requests - 1)
                t = t._replace(positions=t.positions + torch.where(token < t.cu_new[-1:], self.dropped[row], 0))
        self.tables, self._cu_q, self._last = t, None if singles else t.cu_new, None
        return t

    def _pools_of(self, layer: int):
        if self.tables is None:
            raise RuntimeError("begin_step comes before write and attend")
        return self.pools[layer, 0], self.pools[layer, 1]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v: bf16 [Hkv, T, D] views of the step's tokens."""
        ops.paged_cache_write(k, v, *self._pools_of(layer), self.tables.slots)
        if self.weights is not None and self._cu_q is not None:
            ops.paged_weights_clear(self.weights[layer], self.tables.slots)

    def attend(self, layer: int, q: torch.Tensor, softmax_scale: float, window: Optional[int] = None, sinks: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q: bf16 [Hq, T, D] view -> bf16 [T, Hq, D]: every new token over what its request has cached up to it (ops.paged_attention; with groups or
        key_weights, where there is no window and a step brings few tokens, ops.shared_prefix_attention).  A step of single tokens adds what they attend to to the keys' weights; one
        with new_lens leaves them to observe, and so does one with a window: its own keys' are 0 until then.  (What keys in pages of several requests have
        received is not kept.)"""
        pools = self._pools_of(layer)
        if q.dim() == 3 and q.shape[1] != self.tables.slots.numel():
            raise ValueError(f"q has {q.shape[1]} rows, the step {self.tables.slots.numel()}")
        if window is None and (self.shared_lens.numel() > 0 or self.weights is not None) and not self._many_rows(q):
            weights = self.weights[layer] if self.weights is not None and self._cu_q is None else None
            together = q.dim() == 3 and q.shape[0] <= 16 * self.pools.shape[3]  # (attention weighs the keys of up to 16 query heads a kv head)
            out = ops.shared_prefix_attention(q, *pools, self.block_table, self._seen_lens, self.shared_lens, self.cu_groups, softmax_scale,
                                              cu_q=self._cu_q, weights=weights if together else None, out=out, joined=self._joined, first=self._held)
            if weights is not None and not together:
                ops.paged_key_weights(q, pools[0], self.block_table, self._seen_lens, softmax_scale, weights, first=self._held, accumulate=True)
            return out
        if self.weights is not None and self._cu_q is None:
            ops.paged_weights_clear(self.weights[layer], self.tables.slots)
        return ops.paged_attention(q, *pools, self.block_table, self._seen_lens, softmax_scale, cu_q=self._cu_q,
                                   window=window, sinks=sinks, out=out)

    def _many_rows(self, q: torch.Tensor) -> bool:
        """Chunks of prompts: the kernel with matrix products' rate takes less time to read shared keys once a request than the other to read them once.
        us, shared / paged, by rows (tokens x query heads of a kv head) a request: 16 of 32 heads over 8 behind 4096 keys 16: 40 / 57, 32: 54 / 57, 48: 83 / 58,
        128: 102 / 66, 2048: 1021 / 519; 4 behind 32768 keys 32: 72 / 91, 48: 92 / 94, 64: 111 / 94, 2048: 1308 / 879; 16 of 14 over 2 behind 4096 28: 28 / 26, 56:
        34 / 26."""
        return self._cu_q is not None and q.dim() == 3 and q.shape[1] * q.shape[0] > 32 * self.max_requests * self.pools.shape[3]

    def _check_weights(self) -> torch.Tensor:
        if self.weights is None:
            raise RuntimeError("key_weights=True makes a cache that knows its keys' weights")
        return self.weights

    def observe(self, layer: int, q: torch.Tensor, softmax_scale: float, last: int = 32, accumulate: bool = False) -> None:
        """Sets the keys' weights of the requests that bring tokens to what the last `last` tokens of each attend to (all of them, where it brings
        fewer); accumulate: on top of what keys in front of those tokens have (ops.paged_key_weights).  q as for attend, behind write.  Keys in pages of
        several requests have none."""
        weights = self._check_weights()
        pools = self._pools_of(layer)
        if last < 1:
            raise ValueError(f"last must be at least 1, got {last}")
        if q.dim() != 3 or q.shape[1] != self.tables.slots.numel():
            raise ValueError(f"q must be [Hq, {self.tables.slots.numel()}, D], got {tuple(q.shape)}")
        cu = self._cu_q
        if cu is not None:
            if self._last is None or self._last[0] != last:
                count = (cu[1:] - cu[:-1]).clamp(max=last)
                starts = torch.cat((cu[:1], torch.cumsum(count, 0, dtype=torch.int32)))
                token = torch.arange(min(self.max_requests * last, q.shape[1]), dtype=torch.int32, device=q.device)
                row = torch.searchsorted(starts[1:], token, right=True).clamp_(max=self.max_requests - 1)
                source = (cu[1:][row] - count[row] + token - starts[row]).clamp_(0, max(q.shape[1] - 1, 0))
                self._last = (last, starts, source)
            cu, q = self._last[1], q.transpose(0, 1).index_select(0, self._last[2]).transpose(0, 1)
        ops.paged_key_weights(q, pools[0], self.block_table, self._seen_lens, softmax_scale, weights[layer], cu_q=cu, first=self._held,
                              accumulate=accumulate)

    def share(self, group: int, tokens: int) -> int:
        """The first `tokens` keys of the group's first row, as many as fill whole pages, become those of all its rows: the others begin behind them, if they
        are empty.  The first row must have them cached; it may go on as a request of its own, and its end is the end of the sharing (release).  -> how many
        they are: the tokens from there on are the other rows' own to bring."""
        if not 0 <= group < self.shared_lens.numel():
            raise ValueError(f"there are {self.shared_lens.numel()} groups, no group {group}")
        if not 0 <= tokens <= self.block_table.shape[1] * self.page_size:
            raise ValueError(f"{tokens} tokens are none that a request can have")
        first, end = self._group_starts[group:group + 2]
        whole = tokens // self.page_size * self.page_size
        self.shared_lens[group:group + 1].fill_(whole)
        self._joined[first:first + 1].fill_(whole)
        self._held[first:first + 1].clamp_(min=whole)
        # (keys in front of all that evictions have taken stand where they stood in the prompt)
        self._shared_dropped[group:group + 1].copy_(self.dropped[first:first + 1] * (self._in_place[first:first + 1] < whole))
        rows = torch.zeros(self.max_requests, dtype=torch.bool, device=self.lens.device)
        rows[first + 1:end] = True
        self.join(rows)
        return whole

    def join(self, rows: torch.Tensor) -> None:
        """Rows (bool [max_requests]) that are empty, as release leaves them, begin behind what their group shares; others stay as they are, a group's first
        row too.  (An empty row of a group may as well take a request that shares nothing, without joining.)"""
        self._check_mask(rows, "rows")
        # (what an eviction has left nothing of is a request all the same)
        rows = rows & (self.lens == 0) & (self.dropped == 0) & (self._holder != torch.arange(self.max_requests, device=self._holder.device))
        shared = torch.cat((self.shared_lens, self.shared_lens.new_zeros(1)))[self._group_of]
        place = torch.arange(self.block_table.shape[1], device=self.lens.device)[None, :]
        named = torch.where(place * self.page_size < shared[:, None], self.block_table[self._holder], -1)
        self.block_table.copy_(torch.where(rows[:, None], named, self.block_table))
        for x in (self.lens, self._held, self._joined):
            x.copy_(torch.where(rows, shared, x))
        self.dropped.copy_(torch.where(rows & (shared > 0), self._shared_dropped[self._group_of], self.dropped))

    def evict(self, budget: int, recent: int, sinks: int = 0, rows: Optional[torch.Tensor] = None) -> None:
        """Drops keys of requests (rows bool [max_requests]; None: all) that hold more than they may, in every layer and kv head by itself: the first
        `sinks` and those in pages of several requests stay, the last `recent`, and of the others the `budget` heaviest (ops.paged_evict).  Their pages go back.
        A window of attend counts places in the cache, which later keys of such a request have nearer to each other than their positions.
        A request whose rows could not be moved (ops.paged_evict: a length of -1) has its first keys alone, and lost[r] until its release."""
        weights = self._check_weights()
        if rows is not None:
            self._check_mask(rows, "rows")
        lens = self.lens if rows is None else self.lens * rows
        first = torch.clamp(self._held, min=sinks)
        left = torch.stack([ops.paged_evict(*self.pools[layer].unbind(0), weights[layer], self.block_table, lens, budget, recent, first=first)
                            for layer in range(self.pools.shape[0])]).amin(0)
        lost = left < 0
        self.lost |= lost
        left = torch.where(lost, torch.minimum(first, lens), left)
        if rows is not None:
            left = torch.where(rows, left, self.lens)
        in_front = torch.where(self.dropped > 0, torch.minimum(self._in_place, first), first)
        self._in_place.copy_(torch.where(left < self.lens, in_front, self._in_place))
        self.dropped += self.lens - left
        self.lens.copy_(left)
        place = torch.arange(self.block_table.shape[1], device=left.device)[None, :]
        self._give_back(place * self.page_size >= left[:, None])

    def _give_back(self, entries: torch.Tensor) -> None:
        """Puts the pages of entries of the block table (bool, its shape) back on the stack, those that no other entry names, each once."""
        back = entries & (self.block_table >= 0)
        if self.shared_lens.numel() > 0:
            page = torch.where(self.block_table >= 0, self.block_table, self.num_pages).reshape(-1).long()
            kept = torch.zeros(self.num_pages + 1, dtype=torch.bool, device=page.device)
            kept[torch.where(entries.reshape(-1), self.num_pages, page)] = True
            place = torch.arange(page.numel(), device=page.device)
            first = torch.full((self.num_pages + 1,), page.numel(), dtype=torch.int64, device=page.device)
            first.scatter_reduce_(0, torch.where(back.reshape(-1), page, self.num_pages), place, "amin")
            back &= (~kept[page] & (first[page] == place)).reshape(back.shape)
        count = torch.cumsum(back.reshape(-1), 0, dtype=torch.int32)
        place = torch.where(back.reshape(-1), self.free_count + count - 1, self.num_pages)
        self._stack[place.long()] = self.block_table.reshape(-1)
        self.free_count += count[-1:]
        self.block_table.masked_fill_(entries, -1)

    def release(self, finished: torch.Tensor) -> None:
        """Puts the pages of the requests with finished[r] (bool [max_requests]) back on the stack, but for those that others share; their rows are empty
        again.  Where a group's first row finishes its rows share no longer.  Not for a captured graph."""
        self._check_mask(finished, "finished")
        self._give_back(finished[:, None].expand_as(self.block_table))
        self.lens.masked_fill_(finished, 0)
        if self.weights is not None or self.shared_lens.numel() > 0:  # (else they stay 0)
            for x in (self.dropped, self._held, self._joined, self.lost):
                x.masked_fill_(finished, 0)
        if self.shared_lens.numel() > 0:
            ended = finished[self.cu_groups[:-1].long()]
            self.shared_lens.masked_fill_(ended, 0)
            self._shared_dropped[:-1].masked_fill_(ended, 0)
            self._joined.masked_fill_(finished[self._holder], 0)
