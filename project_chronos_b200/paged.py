"""Paged key-value cache of one attention layer for a ragged batch.

``HybridCache`` (``model``) holds contiguous caches whose rows all stand at the
same position.  ``PagedCache`` serves rows of different lengths: each row's slots
lie in pages of ``page_size`` slots taken from one pool, named by the row of a
page table, so memory follows the tokens a row really has.  Keys are stored
rotated, which makes attention independent of the order of the slots and lets
``evict`` cut a row down to a budget by moving only the slots that have to move.

    cache = PagedCache(batch, pages, kv_heads, head_dim, table_width, device, dtype, track_weights=True)
    cache.reserve(row, slots)                       # host: pages for a row
    out = ops.window_attention(q, k, v, cu)         # a packed batch of prompts
    cache.append(k, v, cu)                          # ... into the pages
    cache.append(k1, v1)                            # one token per row (idle rows: with offsets, none)
    out = cache.attend(q1)                          # attention of those tokens
    cache.evict(budget, sinks=4, recent=256)        # least attention goes

The kernels behind it are ``ops.paged_append``, ``ops.paged_attn_decode`` and
``ops.paged_evict`` (include/chronos_paged.h).  append, attend and evict run on
the current stream, read lengths on the device and copy nothing to the host (but
for a window asked for after an eviction, see attend); attend can be captured in
a CUDA graph and replayed while the rows grow.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import ops


class PagedCache:
    """Pages [num_pages, page_size, kv_heads, head_dim] for ``batch`` rows of at most
    ``table_width`` pages each.

    ``lens`` int32 [B]: slots in use; ``seen`` int32 [B]: tokens appended so far (the
    position of the next one).  With ``track_weights``, ``weights`` fp32 and ``positions``
    int32 [B, kv_heads, table_width * page_size] hold every slot's summed attention
    weight and its token's position (``evict`` needs them)."""

    def __init__(self, batch: int, num_pages: int, kv_heads: int, head_dim: int, table_width: int, device,
                 dtype=torch.bfloat16, page_size: int = 64, track_weights: bool = False):
        if min(batch, num_pages, kv_heads, head_dim, table_width, page_size) < 1:
            raise ValueError("batch, num_pages, kv_heads, head_dim, table_width and page_size must be at least 1")
        self.batch, self.num_pages, self.page_size, self.table_width = batch, num_pages, page_size, table_width
        shape = (num_pages, page_size, kv_heads, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        # a page number that is none: its slots are refused, not read
        self.page_table = torch.full((batch, table_width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)
        self.weights: Optional[torch.Tensor] = None
        self.positions: Optional[torch.Tensor] = None
        if track_weights:
            slots = (batch, kv_heads, table_width * page_size)
            self.weights = torch.zeros(slots, dtype=torch.float32, device=device)
            self.positions = torch.zeros(slots, dtype=torch.int32, device=device)
        self._evicted = False    # since the rows were last seen uncut
        self._replays = False    # an eviction was captured: a graph may run it at any time
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch)]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_pages, self.v_pages, self.weights, self.positions)
                   if t is not None)

    def free_pages(self) -> int:
        return len(self._free)

    def _pages_of(self, slots: int) -> int:
        if slots < 0:
            raise ValueError(f"slots must not be negative, got {slots}")
        return -(-int(slots) // self.page_size)

    def reserve(self, row: int, slots: int) -> None:
        """Give ``row`` the pages it lacks for ``slots`` slots (host bookkeeping and one
        copy of its table row)."""
        have = self._pages[row]
        need = self._pages_of(slots)
        if need > self.table_width:
            raise RuntimeError(f"{slots} slots need {need} pages, a row has at most {self.table_width}")
        if need - len(have) > len(self._free):
            raise RuntimeError(f"out of pages: {need - len(have)} needed, {len(self._free)} free")
        if need > len(have):
            have.extend(self._free.pop() for _ in range(need - len(have)))
            self._write_row(row)

    def trim(self, row: int, slots: int) -> None:
        """Give back the pages of ``row`` behind its first ``slots`` slots (after an
        eviction to at most that many: the caller knows the budget).  What lies in them
        is lost: a longer row is cut to the pages it keeps."""
        keep = self._pages_of(slots)
        gone = self._pages[row][keep:]
        if gone:
            del self._pages[row][keep:]
            self._free.extend(reversed(gone))
            self._write_row(row)
            self.lens[row].clamp_(max=keep * self.page_size)

    def release(self, row: int) -> None:
        """End ``row``'s sequence: its pages return to the pool, its length becomes 0."""
        self.trim(row, 0)
        self.lens[row] = 0
        self.seen[row] = 0

    def _write_row(self, row: int) -> None:
        pages = self._pages[row]
        line = torch.tensor(pages + [-1] * (self.table_width - len(pages)), dtype=torch.int32)
        self.page_table[row].copy_(line)

    def append(self, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None) -> None:
        """Append one token per row (k, v [B, kv_heads, D]) or packed sequences
        (``cu_seqlens`` int32 [B + 1]; no tokens for a row that is idle).  A row whose
        pages do not reach drops the tokens behind them, does not count them and records
        CHRONOS_ERR_INVALID_ARG in the status word."""
        ops.paged_append(k, v, self.k_pages, self.v_pages, self.page_table, self.lens, cu_seqlens=cu_seqlens,
                         seen=self.seen, weights=self.weights, positions=self.positions, lens_out=self.lens,
                         seen_out=self.seen)

    def attend(self, q: torch.Tensor, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
               out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each row's newest token (already appended) over its slots, q
        [B, heads, D] -> [B, heads, D]; adds to ``weights`` where they are tracked.
        A window counts slots: it is refused while a row lives that an eviction has cut
        (after an eviction a call with a window reads that from the device, once if no row
        was cut; a graph that was captured with a window must not be replayed then)."""
        if window and (self._evicted or self._replays):
            self._refuse_cut_rows()
        return ops.paged_attn_decode(q, self.k_pages, self.v_pages, self.page_table, self.lens, scale=scale,
                                     window=window, sinks=sinks, weights=self.weights, out=out, lse=lse)

    def _refuse_cut_rows(self) -> None:
        if self.lens.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a window cannot be captured after an eviction: it counts slots, which may be reordered")
        lens, seen = torch.stack([self.lens, self.seen]).tolist()
        cut = [row for row in range(self.batch) if lens[row] != seen[row]]
        if cut:
            raise RuntimeError(f"a window counts slots, which an eviction has reordered in rows {cut}: attend without one")
        self._evicted = False

    def evict(self, budget: int, sinks: int = 0, recent: int = 0) -> torch.Tensor:
        """Cut every row and kv head down to ``budget`` slots (``ops.paged_evict``), in
        place.  Returns src int32 [B, kv_heads, budget]: where each slot came from."""
        if self.weights is None:
            raise RuntimeError("evict needs a cache with track_weights=True")
        src = ops.paged_evict(self.k_pages, self.v_pages, self.page_table, self.lens, self.seen, self.weights,
                              self.positions, budget, sinks=sinks, recent=recent, lens_out=self.lens)["src"]
        self._evicted = True
        self._replays = self._replays or torch.cuda.is_current_stream_capturing()
        return src
