"""A cache of keys and values for answering: pages shared by all layers, rows held in 4 bits, attention over them.

    table = PageTable(requests=16, tokens_per_request=40000, pages=6000, page_size=64, device="cuda:0")
    layers = [KV4Cache(table, kv_heads=4, head_dim=128, dtype=torch.bfloat16) for _ in range(28)]
    # every step: room for the new tokens once, then in each layer
    slots = table.reserve(counts, tokens)
    counts = table.granted(counts, slots)
    cache.append(k, v, slots)
    out = cache.attend(q, counts)

Nothing here reads a length back to the host, so a step can be captured in a CUDA graph and replayed; ops.check_status() says
afterwards whether a request ran out of pages, and `granted` which: its rows come out as zeros."""
from __future__ import annotations

from typing import Optional

import torch

from . import ops


class PageTable:
    """Which pages each request holds, how many tokens it has, and which pages are free (int32 tensors on the device)."""

    def __init__(self, requests: int, tokens_per_request: int, pages: int, page_size: int = 64, device="cuda"):
        if requests < 1 or tokens_per_request < 1 or pages < 1 or page_size < 16 or page_size % 16:
            raise ValueError(f"PageTable: {requests} requests of {tokens_per_request} tokens on {pages} pages of {page_size} (a multiple of 16)")
        self.page_size = page_size
        self.table = torch.full((requests, -(-tokens_per_request // page_size)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.pool = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free = torch.tensor([pages], dtype=torch.int32, device=device)
        ops._need_cuda(self.table)
        ops.status_word(self.table.device)       # before any capture

    @property
    def pages(self) -> int:
        return self.pool.numel()

    def reserve(self, counts: torch.Tensor, tokens: int) -> torch.Tensor:
        """Room for counts[b] <= tokens more tokens of every request -> slots int32 [requests, tokens] (ops.plan_pages, in place).  A request
        that the pool or its row of the table has no room for gets none (see granted)."""
        state = self.table, self.lengths, self.free
        return ops.plan_pages(self.table, self.lengths, counts, self.pool, self.free, self.page_size, tokens, out=state)[3]

    def granted(self, counts: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
        """How many new tokens each request has after reserve(counts, tokens) -> slots: counts, and 0 where it was refused (int32 [requests], on
        the device).  With its own count a refused request's queries would stand at the tokens that it had before."""
        return torch.where(slots[:, 0] >= 0, counts, 0).to(torch.int32)

    def release(self, which: torch.Tensor) -> None:
        """Ends the requests marked in which (bool [requests]): their pages are free again, their lengths 0."""
        ops.release_pages(self.table, self.lengths, which, self.pool, self.free, self.page_size)


class KV4Cache:
    """Keys and values of one layer in 4 bits, on the pages of a PageTable.  group: channels that share a step and a lowest value (32: 5 bits a
    value in all, 64: 4.5, 128: 4.25)."""

    def __init__(self, table: PageTable, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, group: int = 32):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"KV4Cache: float16 or bfloat16, got {dtype}")
        self.table, self.head_dim, self.dtype, self.group = table, head_dim, dtype, group
        self.data = ops.kv4_empty(table.pages, kv_heads, table.page_size, head_dim, group, table.table.device)

    def _own(self, x: torch.Tensor) -> None:
        if x.dtype != self.dtype or x.shape[-1] != self.head_dim:
            raise ValueError(f"a cache of {self.dtype} rows of {self.head_dim} channels, got {x.dtype} rows of {x.shape[-1]}")

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Rows k, v [requests, kv_heads, tokens, head_dim] into the slots that PageTable.reserve gave (ops.kv4_append)."""
        self._own(k), self._own(v)
        ops.kv4_append(self.data, k, v, slots, self.group)

    def read(self, slots: torch.Tensor):
        """What slots [B, n] hold, as keys and values [B, kv_heads, n, head_dim] (ops.kv4_read)."""
        return ops.kv4_read(self.data, slots, self.head_dim, self.group, self.dtype)

    def attend(self, q: torch.Tensor, counts: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None, return_lse: bool = False):
        """Attention of the newest tokens q [requests, heads, tokens, head_dim], their keys appended before (ops.kv4_attention); counts: as
        PageTable.granted gives them."""
        self._own(q)
        return ops.kv4_attention(q, self.data, self.table.table, self.table.lengths, self.group, counts, sm_scale, return_lse)
