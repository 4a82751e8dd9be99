"""A key / value cache in pages for serving: pools, block tables and a stack of unused pages, all on the GPU.

    cache = PagedKVCache(num_layers=32, num_pages=4096, num_kv_heads=8, head_dim=128, max_requests=16, max_tokens=131072)
    cache.begin_step(new_lens, max_new_tokens=512)          # tokens each request brings (0: none): prompts in chunks, next tokens
    for layer in range(32):                                 # q, k, v of the step's tokens, request after request
        cache.write(layer, k, v)
        out = cache.attend(layer, q, softmax_scale)
    cache.begin_step(active=running)                        # a token of each running request, rows request by request
    cache.release(finished)

A step (begin_step, write, attend) reads no device value on the host, so it can be recorded into a HIP graph and replayed with other lengths;
release runs between steps.  The reference keeps no cache of its own (its decode step reads a contiguous one, shareprefill_attn.py:146-155).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops


class PagedKVCache:
    """Requests are rows 0 .. max_requests - 1 of the block table; one model runs its steps in order on one stream."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, max_requests: int, max_tokens: int,
                 page_size: int = 64, device="cuda"):
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
        (negative: they did not; tokens without a slot are not cached and seen by nobody)."""
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
        self.tables, self._cu_q = t, None if singles else t.cu_new
        return t

    def _pools_of(self, layer: int):
        if self.tables is None:
            raise RuntimeError("begin_step comes before write and attend")
        return self.pools[layer, 0], self.pools[layer, 1]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v: bf16 [Hkv, T, D] views of the step's tokens."""
        ops.paged_cache_write(k, v, *self._pools_of(layer), self.tables.slots)

    def attend(self, layer: int, q: torch.Tensor, softmax_scale: float, window: Optional[int] = None, sinks: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q: bf16 [Hq, T, D] view -> bf16 [T, Hq, D]: every new token over what its request has cached up to it (ops.paged_attention)."""
        pools = self._pools_of(layer)
        if q.dim() == 3 and q.shape[1] != self.tables.slots.numel():
            raise ValueError(f"q has {q.shape[1]} rows, the step {self.tables.slots.numel()}")
        return ops.paged_attention(q, *pools, self.block_table, self._seen_lens, softmax_scale, cu_q=self._cu_q,
                                   window=window, sinks=sinks, out=out)

    def release(self, finished: torch.Tensor) -> None:
        """Puts the pages of the requests with finished[r] (bool [max_requests]) back on the stack; their rows are empty again.
        Not for a captured graph."""
        self._check_mask(finished, "finished")
        back = finished[:, None] & (self.block_table >= 0)
        count = torch.cumsum(back.reshape(-1), 0, dtype=torch.int32)
        place = torch.where(back.reshape(-1), self.free_count + count - 1, self.num_pages)
        self._stack[place.long()] = self.block_table.reshape(-1)
        self.free_count += count[-1:]
        self.block_table.masked_fill_(finished[:, None], -1)
        self.lens.masked_fill_(finished, 0)
