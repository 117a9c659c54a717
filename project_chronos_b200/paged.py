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

    cache = PagedCache(..., four_bit=True, page_bounds=True)
    q = cache.append_rope(q, k, v, cos, sin)        # rotated on the way into pages of 4-bit values
    out = cache.attend(q)                           # ... over all of a row
    out, pages = cache.attend_sparse(q, topk=32)    # ... over the pages that score highest
    k, v = cache.gather(cu, rows)                   # rows of the cache, for prompt attention

The kernels behind it are ``ops.paged_append``, ``ops.paged_attn_decode`` and
``ops.paged_evict`` (include/chronos_paged.h), ``ops.paged_append_rope``,
``ops.paged_attn_decode4``, ``ops.paged_gather``, ``ops.paged_bounds``,
``ops.paged_select`` and ``ops.paged_attn_sparse`` (include/chronos_paged4.h).  All of them
run on the current stream, read lengths on the device and copy nothing to the host (but
for a window asked for after an eviction, see attend); they can be captured in
a CUDA graph and replayed while the rows grow.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import ops


class PagedCache:
    """Pages [num_pages, page_size, kv_heads, head_dim] for ``batch`` rows of at most
    ``table_width`` pages each.

    ``lens`` int32 [B]: slots in use; ``seen`` int32 [B]: tokens appended so far (the
    position of the next one).  With ``track_weights``, ``weights`` fp32 and ``positions``
    int32 [B, kv_heads, table_width * page_size] hold every slot's summed attention
    weight and its token's position (``evict`` needs them).

    With ``four_bit`` the pages hold 4-bit values in units of ``k_scale`` and ``v_scale`` (uint8
    [num_pages, kv_heads, bytes], 9 bytes for 16 columns; page_size a multiple of 16).  With
    ``page_bounds``, ``bounds`` [num_pages, 2, kv_heads, head_dim] are the smallest and largest
    key of every page, which the appends keep up to date (``attend_sparse`` needs them).  Neither
    goes with ``track_weights``: what an eviction moves is not 4 bits, and leaves its page's
    bounds behind."""

    def __init__(self, batch: int, num_pages: int, kv_heads: int, head_dim: int, table_width: int, device,
                 dtype=torch.bfloat16, page_size: int = 64, track_weights: bool = False, four_bit: bool = False,
                 page_bounds: bool = False, k_scale: float = 1.0, v_scale: float = 1.0):
        if min(batch, num_pages, kv_heads, head_dim, table_width, page_size) < 1:
            raise ValueError("batch, num_pages, kv_heads, head_dim, table_width and page_size must be at least 1")
        if track_weights and (four_bit or page_bounds):
            raise ValueError("track_weights goes neither with four_bit nor with page_bounds")
        self.batch, self.num_pages, self.page_size, self.table_width = batch, num_pages, page_size, table_width
        self.kv_heads, self.head_dim, self.dtype, self.four_bit = kv_heads, head_dim, dtype, four_bit
        self.k_scale, self.v_scale = (k_scale, v_scale) if four_bit else (1.0, 1.0)
        shape = (num_pages, page_size, kv_heads, head_dim)
        if four_bit:
            shape = (num_pages, kv_heads, ops.packed_page_bytes(page_size, head_dim))
        self.k_pages = torch.zeros(shape, dtype=torch.uint8 if four_bit else dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=torch.uint8 if four_bit else dtype, device=device)
        self.bounds: Optional[torch.Tensor] = None
        if page_bounds:
            self.bounds = torch.zeros((num_pages, 2, kv_heads, head_dim), dtype=dtype, device=device)
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
        return sum(t.numel() * t.element_size() for t in (self.k_pages, self.v_pages, self.weights, self.positions,
                                                                  self.bounds) if t is not None)

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
        if self.four_bit:
            ops.paged_append_rope(k, v, self.k_pages, self.v_pages, self.page_table, self.lens, self.seen,
                                  cu_seqlens=cu_seqlens, lens_out=self.lens, seen_out=self.seen, k_scale=self.k_scale,
                                  v_scale=self.v_scale)
        else:
            ops.paged_append(k, v, self.k_pages, self.v_pages, self.page_table, self.lens, cu_seqlens=cu_seqlens,
                             seen=self.seen, weights=self.weights, positions=self.positions, lens_out=self.lens,
                             seen_out=self.seen)
        self._update_bounds(k.shape[0], cu_seqlens)

    def append_rope(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                    cu_seqlens: Optional[torch.Tensor] = None, rope_start: int = 0, q_out: Optional[torch.Tensor] = None,
                    k_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """``append`` of rows that are not rotated yet: keys and queries (q [T, heads, D] or
        None) turn by the angles of their positions (``seen`` on), cos and sin [positions, R].
        Returns the rotated queries (``q_out``, which may be q); ``k_out`` (may be k) receives the
        rotated keys.  A position behind the tables drops the token like a missing page."""
        q_out = ops.paged_append_rope(k, v, self.k_pages, self.v_pages, self.page_table, self.lens, self.seen, cos, sin,
                                      q=q, q_out=q_out, k_out=k_out, cu_seqlens=cu_seqlens, rope_start=rope_start,
                                      weights=self.weights, positions=self.positions, lens_out=self.lens,
                                      seen_out=self.seen, k_scale=self.k_scale, v_scale=self.v_scale)
        self._update_bounds(k.shape[0], cu_seqlens)
        return q_out

    def _update_bounds(self, tokens: int, cu_seqlens: Optional[torch.Tensor]) -> None:
        if self.bounds is not None:
            ops.paged_bounds(self.k_pages, self.bounds, self.page_table, self.lens, cu_seqlens=cu_seqlens,
                             num_tokens=tokens, k_scale=self.k_scale)

    def gather(self, cu_seqlens: torch.Tensor, rows: int, first: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of the cache as packed rows [rows, kv_heads, D]: cu_seqlens[b] + i is
        slot first[b] + i of row b (default: its newest cu_seqlens[b + 1] - cu_seqlens[b] slots).
        Rows behind the last sequence are zeros."""
        shape = (rows, self.kv_heads, self.head_dim)
        k, v = (torch.zeros(shape, dtype=self.dtype, device=self.k_pages.device) for _ in range(2))
        return ops.paged_gather(self.k_pages, self.v_pages, self.page_table, self.lens, cu_seqlens, k, v, first=first,
                                k_scale=self.k_scale, v_scale=self.v_scale)

    def attend(self, q: torch.Tensor, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
               out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each row's newest token (already appended) over its slots, q
        [B, heads, D] -> [B, heads, D]; adds to ``weights`` where they are tracked.
        A window counts slots: it is refused while a row lives that an eviction has cut
        (after an eviction a call with a window reads that from the device, once if no row
        was cut; a graph that was captured with a window must not be replayed then)."""
        if self.four_bit:
            return ops.paged_attn_decode4(q, self.k_pages, self.v_pages, self.page_table, self.lens, scale=scale,
                                          window=window, sinks=sinks, k_scale=self.k_scale, v_scale=self.v_scale,
                                          out=out, lse=lse)
        if window and (self._evicted or self._replays):
            self._refuse_cut_rows()
        return ops.paged_attn_decode(q, self.k_pages, self.v_pages, self.page_table, self.lens, scale=scale,
                                     window=window, sinks=sinks, weights=self.weights, out=out, lse=lse)

    def attend_sparse(self, q: torch.Tensor, topk: int, first: int = 1, last: int = 2, scale: Optional[float] = None,
                      cu_seqlens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                      lse: Optional[torch.Tensor] = None, pages: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Attention over ``topk`` pages per token and kv head: the ``first`` ones, the ``last`` ones
        up to its own, and the others whose keys may score highest.  q [B, heads, D] of each
        row's newest token, or [T, heads, D] of its newest ones with ``cu_seqlens`` (already
        appended).  Returns (out, pages int32 [T, kv_heads, topk])."""
        if self.bounds is None:
            raise RuntimeError("attend_sparse needs a cache with page_bounds=True")
        pages = ops.paged_select(q, self.bounds, self.page_table, self.lens, self.page_size, topk, first=first, last=last,
                                 cu_seqlens=cu_seqlens, out=pages)
        out = ops.paged_attn_sparse(q, self.k_pages, self.v_pages, self.page_table, self.lens, pages, cu_seqlens=cu_seqlens,
                                    scale=scale, k_scale=self.k_scale, v_scale=self.v_scale, out=out, lse=lse)
        return out, pages

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
