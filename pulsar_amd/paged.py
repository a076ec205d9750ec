"""A paged key-value cache for the layers of a model, over the operators of pulsar_amd.ops.

The pool holds keys and values of every layer as planes of one tensor, [2 * layers, pages,
page_size, kv_heads, head_dim], so a page id names the same page in all of them and forking, copying
and compacting are one call for the whole model.  The book-keeping -- reference counts, block tables,
lengths -- is on the device and changes in place; the host keeps only an upper bound of each row's
length, which sizes the attention's grid.  No method but `lengths` waits for the device.  Methods that
take lists copy them to the device when they are called, so they do not belong into a captured graph;
the operators may.

The reference's engine holds such a pool behind its attention (pulsar-core's ActiveBuffer,
active_buffer.hpp:164, and the scatter of new keys at paged_attention.cu:48).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops


@dataclass
class Step:
    """The new tokens of one call of a model: `counts[b]` of row b, row after row.  `missing` (int32
    [1] on the device) is 0 where the pool had room for them; else nothing was taken, and the step's
    tokens are not stored."""
    counts: list[int]
    cu_q: torch.Tensor
    slots: torch.Tensor
    missing: torch.Tensor
    max_q_len: int
    max_seq_len: int


class PagedKVCache:
    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, rows: int,
                 max_seq_len: int, dtype: torch.dtype = torch.bfloat16, device="cuda:0"):
        if min(layers, pages, page_size, kv_heads, head_dim, rows, max_seq_len) <= 0:
            raise ValueError("PagedKVCache: every size must be positive")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"PagedKVCache: dtype must be fp16 or bf16, got {dtype}")
        self.page_size, self.rows = page_size, rows
        self.pool = torch.empty((2 * layers, pages, page_size, kv_heads, head_dim), dtype=dtype, device=device)
        ints = {"dtype": torch.int32, "device": device}
        self.ref_counts = torch.zeros(pages, **ints)
        self.block_tables = torch.full((rows, -(-max_seq_len // page_size)), -1, **ints)
        self.seq_lens = torch.zeros(rows, **ints)
        self._most = [0] * rows  # at most so many tokens in each row

    def layer(self, index: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a layer, [pages, page_size, kv_heads, head_dim]."""
        return self.pool[2 * index], self.pool[2 * index + 1]

    def _ints(self, values: list[int]) -> torch.Tensor:
        # Pageable memory: such a copy of up to 4096 rows' numbers returns at once, the device busy or
        # not, as a test holds it to, and 3 us sooner than one from pinned memory.
        return torch.tensor(values, dtype=torch.int32).to(self.seq_lens.device, non_blocking=True)

    def extend(self, counts: list[int]) -> Step:
        """Takes pages for counts[b] new tokens of row b."""
        if len(counts) != self.rows or min(counts) < 0:
            raise ValueError(f"PagedKVCache.extend: {self.rows} counts of new tokens, got {counts}")
        total = [0]
        for c in counts:
            total.append(total[-1] + c)
        cu_q = self._ints(total)
        slots, missing = ops.paged_cache_extend(self.ref_counts, self.block_tables, self.seq_lens, cu_q, total[-1],
                                                self.page_size)
        most = self.block_tables.shape[1] * self.page_size  # an extend past a row's table is refused
        self._most = [min(m + c, most) for m, c in zip(self._most, counts)]
        seen = [m for m, c in zip(self._most, counts) if c]
        return Step(list(counts), cu_q, slots, missing, max(counts), max(seen, default=0))

    def lengths(self) -> list[int]:
        """Each row's tokens, read from the device: this waits for it.  The host's bounds of the rows are
        exact afterwards.  (They only grow else until a row is freed, also by what a full pool refused;
        a bound that is too high costs speed, not results.)"""
        self._most = self.seq_lens.tolist()
        return list(self._most)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: Step) -> None:
        """Stores the step's keys and values [T, kv_heads, head_dim] of a layer."""
        ops.paged_cache_write(k, v, *self.layer(layer), step.slots)

    def attend(self, layer: int, q: torch.Tensor, step: Step, **options):
        """Attention of the step's queries [T, q_heads, head_dim] over their rows, with the options of
        ops.paged_attention."""
        return ops.paged_attention(q, *self.layer(layer), self.block_tables, self.seq_lens, step.cu_q, step.max_q_len,
                                   step.max_seq_len, **options)

    def _rows(self, rows: list[int], what: str) -> torch.Tensor:
        if any(not 0 <= r < self.rows for r in rows):
            raise ValueError(f"PagedKVCache.{what}: rows are 0 to {self.rows - 1}, got {rows}")
        return self._ints(rows)

    def fork(self, src: list[int], dst: list[int]) -> torch.Tensor:
        """Rows dst become copies of rows src; returns the free pages that lacked (int32 [1]).  What the
        rows dst held is given back first, whether or not there is room for the copies."""
        if len(src) != len(dst) or len(set(dst)) != len(dst) or set(src) & set(dst):
            raise ValueError("PagedKVCache.fork: as many sources as destinations, each destination once and no source")
        src_rows, dst_rows = self._rows(src, "fork"), self._rows(dst, "fork")
        if any(self._most[d] for d in dst):
            ops.paged_cache_free(self.ref_counts, self.block_tables, self.seq_lens, dst_rows)
        missing = ops.paged_cache_fork(self.pool, self.ref_counts, self.block_tables, self.seq_lens, src_rows, dst_rows)
        for s, d in zip(src, dst):
            self._most[d] = self._most[s]
        return missing

    def free(self, rows: list[int]) -> None:
        ops.paged_cache_free(self.ref_counts, self.block_tables, self.seq_lens, self._rows(rows, "free"))
        for r in rows:
            self._most[r] = 0

    def compact(self) -> torch.Tensor:
        """Moves the pages in use to the pool's start; returns how many there are (int32 [1])."""
        return ops.paged_cache_compact(self.pool, self.ref_counts, self.block_tables)
