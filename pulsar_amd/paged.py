"""A paged key-value cache for the layers of a model, over the operators of pulsar_amd.ops.

The pool holds keys and values of every layer as planes of one tensor, [2 * layers, pages,
page_size, kv_heads, head_dim] (with bits=4 bytes, the last dimension head_dim / 2 + head_dim / 32), so
a page id names the same page in all of them and forking, copying and compacting are one call for the
whole model.  The book-keeping -- reference counts, block tables,
lengths -- is on the device and changes in place; the host keeps only an upper bound of each row's
length, which sizes the attention's grid.  No method but `lengths` waits for the device, and `append` where
that bound does not tell whether its table of rotations is long enough.  Methods that
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
    positions: torch.Tensor | None = None  # of the tokens, int64: PagedKVCache.positions
    changes: int = -1  # the cache's, when the step was taken
    reach: int | None = None  # positions that its stored tokens need of a table: read where max_seq_len is too high


class PagedKVCache:
    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, rows: int,
                 max_seq_len: int, dtype: torch.dtype = torch.bfloat16, device="cuda:0", bits: int = 16):
        if min(layers, pages, page_size, kv_heads, head_dim, rows, max_seq_len) <= 0:
            raise ValueError("PagedKVCache: every size must be positive")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"PagedKVCache: dtype must be fp16 or bf16, got {dtype}")
        if bits not in (4, 16) or (bits == 4 and (head_dim % 32 or head_dim > 256)):
            raise ValueError(f"PagedKVCache: bits must be 16, or 4 with head_dim a multiple of 32 up to 256, got {bits}")
        self.page_size, self.rows, self.bits, self.dtype = page_size, rows, bits, dtype
        if bits == 16:
            self.pool = torch.empty((2 * layers, pages, page_size, kv_heads, head_dim), dtype=dtype, device=device)
        else:
            row = head_dim // 2 + head_dim // 32
            size = page_size * kv_heads * row  # a page's; pages begin at multiples of 16
            flat = torch.empty((2 * layers, pages, -(-size // 16) * 16), dtype=torch.uint8, device=device)
            self.pool = flat[:, :, :size].unflatten(2, (page_size, kv_heads, row))
        ints = {"dtype": torch.int32, "device": device}
        self.ref_counts = torch.zeros(pages, **ints)
        self.block_tables = torch.full((rows, -(-max_seq_len // page_size)), -1, **ints)
        self.seq_lens = torch.zeros(rows, **ints)
        self._most = [0] * rows  # at most so many tokens in each row
        self._changes = 0  # calls that may have changed a row's length

    def layer(self, index: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a layer, [pages, page_size, kv_heads, head_dim] (bytes with bits=4)."""
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
        self._changes += 1
        return Step(list(counts), cu_q, slots, missing, max(counts), max(seen, default=0), changes=self._changes)

    def lengths(self) -> list[int]:
        """Each row's tokens, read from the device: this waits for it.  The host's bounds of the rows are
        exact afterwards.  (They only grow else until a row is freed, also by what a full pool refused;
        a bound that is too high costs speed, not results.)"""
        self._most = self.seq_lens.tolist()
        return list(self._most)

    def _check(self, x: torch.Tensor, what: str) -> None:
        # 4 bits hold magnitudes of bf16 that fp16 has not, and do not know which they are of
        if self.bits == 4 and x.dtype != self.dtype:
            raise ValueError(f"PagedKVCache.{what}: the cache is of {self.dtype}, got {x.dtype}")

    def positions(self, step: Step) -> torch.Tensor:
        """The positions of a step's tokens in their rows, int64 [T], made once a step from the rows' lengths:
        before the next step, and before rows are forked, reordered or freed."""
        if step.positions is None:
            if step.changes != self._changes:
                raise ValueError("PagedKVCache.positions: the rows have changed since the step was taken")
            n = step.cu_q[1:] - step.cu_q[:-1]
            tokens = step.slots.shape[0]
            row = torch.repeat_interleave(n, output_size=tokens)
            # (a step that was refused has the positions it would have had, and no slots)
            first = self.seq_lens - torch.where(step.missing == 0, n, 0) - step.cu_q[:-1]
            step.positions = torch.arange(tokens, device=row.device) + first[row]
        return step.positions

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: Step) -> None:
        """Stores the step's keys and values [T, kv_heads, head_dim] of a layer."""
        self._check(k, "write")
        if self.bits == 16:
            ops.paged_cache_write(k, v, *self.layer(layer), step.slots)
        else:
            ops.paged_cache_append_fp4(None, k, v, *self.layer(layer), step.slots)

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: Step, rope: torch.Tensor,
               interleaved: bool = False) -> torch.Tensor:
        """Rotates the step's queries and keys by their positions in their rows (ops.paged_cache_append's
        rotation, `rope` of at least as many positions as a row has), stores the keys and values and returns
        the queries.  The step's positions are taken with the first layer.

        A table that ends before a token that would be stored raises ValueError, and nothing is stored.  The
        bound step.max_seq_len tells mostly; where it is above the table's rows the positions are read, once a
        step, which waits for the device (not while a graph is captured: a table is taken as it is there)."""
        self._check(k, "append")
        positions = self.positions(step)
        if rope.dim() == 2 and rope.shape[0] < step.max_seq_len and not torch.cuda.is_current_stream_capturing():
            if step.reach is None:
                stored = torch.where(step.slots >= 0, positions, -1)
                step.reach = 1 + int(stored.max()) if stored.numel() else 0
            if rope.shape[0] < step.reach:
                raise ValueError(f"PagedKVCache.append: rope has {rope.shape[0]} positions, a row {step.reach}")
        append = ops.paged_cache_append if self.bits == 16 else ops.paged_cache_append_fp4
        return append(q, k, v, *self.layer(layer), step.slots, rope, positions, interleaved)

    def attend(self, layer: int, q: torch.Tensor, step: Step, **options):
        """Attention of the step's queries [T, q_heads, head_dim] over their rows, with the options of
        ops.paged_attention."""
        self._check(q, "attend")
        attention = ops.paged_attention if self.bits == 16 else ops.paged_attention_fp4
        return attention(q, *self.layer(layer), self.block_tables, self.seq_lens, step.cu_q, step.max_q_len,
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
        self._changes += 1
        return missing

    def reorder(self, rows: torch.Tensor, live: list[int], spare: list[int]) -> torch.Tensor:
        """Beams go on: row spare[i] becomes a copy of row live[rows[i]], and the rows `live` are given back.
        `rows` is int32 on the device, ops.beam_select's rows where live[j] is what row j of its logits
        belongs to; where one names none of `live`, spare[i] stays empty.  Returns the free pages that lacked
        (int32 [1]), in which case no row changed, but that what the rows `spare` held is given back first."""
        if len(set(spare)) != len(spare) or set(live) & set(spare) or rows.numel() != len(spare):
            raise ValueError("PagedKVCache.reorder: a spare row for each of rows, each once and not live")
        n = len(live)
        ints = self._rows(live + spare, "reorder")
        to_rows = ints[n:]
        # a row outside becomes 0 and so -1, a pair that fork passes over
        from_rows = ops.beam_reorder([ints[:n] + 1], rows)[0] - 1
        if any(self._most[r] for r in spare):
            ops.paged_cache_free(self.ref_counts, self.block_tables, self.seq_lens, to_rows)
        missing = ops.paged_cache_fork(self.pool, self.ref_counts, self.block_tables, self.seq_lens, from_rows, to_rows)
        # nothing goes where nothing was copied: a row below 0 is none
        ops.paged_cache_free(self.ref_counts, self.block_tables, self.seq_lens,
                             torch.sub(ints[:n], missing, alpha=self.rows))
        # (the bounds of `live` stay: the host does not know whether there was room)
        most = max((self._most[r] for r in live), default=0)
        for r in spare:
            self._most[r] = most
        self._changes += 1
        return missing

    def free(self, rows: list[int]) -> None:
        ops.paged_cache_free(self.ref_counts, self.block_tables, self.seq_lens, self._rows(rows, "free"))
        for r in rows:
            self._most[r] = 0
        self._changes += 1

    def compact(self) -> torch.Tensor:
        """Moves the pages in use to the pool's start; returns how many there are (int32 [1])."""
        return ops.paged_cache_compact(self.pool, self.ref_counts, self.block_tables)
