"""Pages of the KV cache: copies, compaction, and page tables on the device.

:class:`CachePages` moves bytes in every layer's pools at once; a program whose
block manager lives on the host (the reference's, or the engine's BlockPool)
uses it as it is.  :class:`PagePool` keeps the block manager's part on the
device as well: reference counts beside a table such as
:class:`mkv.decode_state.DecodeMetadata`'s, so that sequences fork (parallel
samples, beams), grow and are freed without a word from the host.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from . import _lib
from .attention import _block_table, _call_on, _require_gpu, _stream

MAX_ROWS = 1024
MAX_ACCEPTED = 2048


def _index_code(t: torch.Tensor, what: str) -> int:
    if t.dtype == torch.int64:
        return _lib.INDEX_I64
    if t.dtype == torch.int32:
        return _lib.INDEX_I32
    raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")


class CachePages:
    """The paged tensors of a cache, all layers' K and V pools (and, with
    per-token-head formats, their scales): each (num_blocks, block_size, ...),
    contiguous, a multiple of 4 bytes a token, none overlapping another.  The
    tensors are kept; they must stay where they are."""

    def __init__(self, caches: Sequence[torch.Tensor]):
        self.caches = tuple(caches)
        if not self.caches:
            raise ValueError("no cache tensors")
        self.device = _require_gpu(*self.caches)
        shape = self.caches[0].shape[:2]
        if len(shape) != 2 or not all(shape):
            raise ValueError(f"a cache tensor must be (num_blocks, block_size, ...); got {tuple(self.caches[0].shape)}")
        self.num_blocks, self.block_size = shape
        if self.block_size & (self.block_size - 1):
            raise ValueError(f"block_size must be a power of two; got {self.block_size}")
        tokens = self.num_blocks * self.block_size
        ptrs, rows = [], []
        for t in self.caches:
            if t.shape[:2] != shape:
                raise ValueError(f"cache tensors of {tuple(t.shape[:2])} and {tuple(shape)} blocks and rows")
            if not t.is_contiguous():
                raise ValueError("cache tensors must be contiguous")
            ptr, row = t.data_ptr(), t.nbytes // tokens
            if row == 0 or row % 4 or ptr % 4:
                raise ValueError(f"a token's row must be a multiple of 4 bytes; got {tuple(t.shape)} {t.dtype}")
            ptrs.append(ptr)
            rows.append(row)
        spans = sorted(zip(ptrs, rows))
        if any(a + n * tokens > b for (a, n), (b, _) in zip(spans, spans[1:])):
            raise ValueError("cache tensors overlap")
        n = len(ptrs)
        self._ptrs = (ctypes.c_void_p * n)(*ptrs)
        self._rows = (ctypes.c_int64 * n)(*rows)
        self._pools = (ctypes.addressof(self._ptrs), ctypes.addressof(self._rows), n, self.num_blocks, self.block_size)

    def copy(self, src: torch.Tensor | Sequence[int], dst: torch.Tensor | Sequence[int]) -> None:
        """Page src[i] to page dst[i] in every tensor.  No page may be the
        destination of two pairs, or the destination of one and the source of
        another: lists and CPU tensors are checked (as are their ranges), GPU
        tensors (int32 or int64) cannot be; there, pairs that name a page outside
        the pool are skipped."""
        if not (isinstance(src, torch.Tensor) and src.is_cuda and isinstance(dst, torch.Tensor) and dst.is_cuda):
            src, dst = (x.tolist() if isinstance(x, torch.Tensor) else list(x) for x in (src, dst))
            if len(src) != len(dst):
                raise ValueError(f"{len(src)} source and {len(dst)} destination pages")
            if not all(0 <= p < self.num_blocks for p in src + dst):
                raise ValueError(f"a page outside 0..{self.num_blocks - 1}")
            if len(set(dst)) != len(dst) or set(src) & set(dst):
                raise ValueError("a page is the destination of two pairs, or a source and a destination")
            src, dst = torch.tensor([src, dst], dtype=torch.int64).to(self.device)
        _require_gpu(self.caches[0], src, dst)
        if src.dim() != 1 or src.shape != dst.shape:
            raise ValueError(f"src {tuple(src.shape)} and dst {tuple(dst.shape)} must be of one length")
        if src.dtype != dst.dtype:
            raise TypeError(f"src {src.dtype} and dst {dst.dtype} must share a dtype")
        code = _index_code(src, "src")
        src, dst = src.contiguous(), dst.contiguous()
        if src.numel():
            _call_on(self.device, "mkv_copy_pages", *self._pools, src.data_ptr(), dst.data_ptr(), code, src.numel(),
                     _stream(self.device))

    def compact(self, block_tables: torch.Tensor, prefix_lens: torch.Tensor, accepted: torch.Tensor) -> None:
        """Move the accepted drafted tokens' rows up behind the prefix: in
        every tensor, row prefix_lens[b] + accepted[b, j] of sequence b to row
        prefix_lens[b] + j, every row of a sequence read before one is written.

        accepted: int32 or int64 (batch, up to 2048), offsets into the drafted
        tokens; entries below 0, and rows outside the block table or the pool, are
        skipped.  block_tables: int32 (batch or more, blocks).  Sequences must not
        share the pages of these rows."""
        _require_gpu(self.caches[0], block_tables, prefix_lens, accepted)
        if accepted.dim() != 2 or accepted.shape[1] > MAX_ACCEPTED:
            raise ValueError(f"accepted must be (batch, up to {MAX_ACCEPTED}); got {tuple(accepted.shape)}")
        batch, n = accepted.shape
        if block_tables.dim() != 2 or block_tables.shape[0] < batch or prefix_lens.dim() != 1 or prefix_lens.numel() < batch:
            raise ValueError(f"block_tables {tuple(block_tables.shape)} and prefix_lens {tuple(prefix_lens.shape)} "
                             f"must cover {batch} sequences")
        if batch > 65535:
            raise ValueError(f"batch {batch} > 65535")
        bt = _block_table(block_tables)
        codes = _index_code(prefix_lens, "prefix_lens"), _index_code(accepted, "accepted")
        prefix_lens = prefix_lens.contiguous()
        if n and (accepted.stride(1) != 1 or accepted.stride(0) < n):
            accepted = accepted.contiguous()
        if batch and n:
            _call_on(self.device, "mkv_compact_slots", *self._pools, bt.data_ptr(), bt.stride(0), bt.shape[1],
                     prefix_lens.data_ptr(), codes[0], accepted.data_ptr(), codes[1],
                     accepted.stride(0) if batch > 1 else n, batch, n, _stream(self.device))


class PagePool:
    """Reference-counted pages for a table of up to 1024 rows.

    block_tables: int32 (rows, max_blocks), and seq_lens: int64 (rows,), the
    tokens in each row's pages (0: a free row), e.g. those of a
    :class:`mkv.decode_state.DecodeMetadata`; both are changed in place.
    ref_counts (int32, one a page) and held (int32, pages of each row) are made
    empty, for tables without sequences, unless they are given.  A page that the
    pool must not hand out is one with a count of its own (``ref_counts[p] += 1``:
    a prefix that stays cached, say)."""

    def __init__(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, pages: CachePages,
                 ref_counts: torch.Tensor | None = None, held: torch.Tensor | None = None):
        dev = _require_gpu(pages.caches[0], block_tables, seq_lens)
        if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or block_tables.stride(1) != 1:
            raise ValueError("block_tables must be an int32 (rows, max_blocks) tensor with contiguous rows")
        rows, self.max_blocks = block_tables.shape
        if not 0 < rows <= MAX_ROWS or not self.max_blocks or (rows > 1 and block_tables.stride(0) < self.max_blocks):
            raise ValueError(f"block_tables must hold 1..{MAX_ROWS} rows of their own; got {tuple(block_tables.shape)}")
        ref_counts = torch.zeros(pages.num_blocks, dtype=torch.int32, device=dev) if ref_counts is None else ref_counts
        held = torch.zeros(rows, dtype=torch.int32, device=dev) if held is None else held
        _require_gpu(block_tables, ref_counts, held)
        for name, t, n, dtype in (("seq_lens", seq_lens, rows, torch.int64), ("held", held, rows, torch.int32),
                                  ("ref_counts", ref_counts, pages.num_blocks, torch.int32)):
            if t.shape != (n,) or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n}; got {t.dtype} {tuple(t.shape)}")
        self.pages, self.device, self.rows = pages, dev, rows
        self.block_tables, self.seq_lens, self.ref_counts, self.held = block_tables, seq_lens, ref_counts, held

    def assign(self, parents: torch.Tensor, tokens: torch.Tensor | None = None) -> torch.Tensor:
        """One step of the table, on the device: row i goes on with the
        sequence that row parents[i] held before the call (its own where
        parents[i] == i; below 0: it is freed), then grows to pages for
        tokens[i] tokens (of the sequence's whole length; None: no growth).

        Full pages are shared.  A part-filled last page that has other holders is
        copied, its filled rows only, in every cache tensor, for all rows but the
        first.  Fresh pages are the lowest-numbered free ones, handed out in row
        order.  Returns a bool (rows,) tensor: False for a row that was refused
        because the pool or the table has no room (it ends freed, or as it was if
        it went on with its own sequence), or because its parent is not a row.
        Requests are served in row order: pages that a refused row asked for are
        not handed to the rows behind it, which are refused too if they need any.

        parents, tokens: int32 or int64 (rows,).  seq_lens takes the parent's
        length (0 for a row without one: a new request's, set once its prompt is
        in)."""
        _require_gpu(self.block_tables, parents, *(() if tokens is None else (tokens,)))
        for name, t in (("parents", parents), ("tokens", tokens)):
            if t is not None and t.shape != (self.rows,):
                raise ValueError(f"{name} must be ({self.rows},); got {tuple(t.shape)}")
        codes = _index_code(parents, "parents"), 0 if tokens is None else _index_code(tokens, "tokens")
        parents = parents.contiguous()
        tokens = None if tokens is None else tokens.contiguous()
        granted = torch.empty(self.rows, dtype=torch.bool, device=self.device)
        nbytes = _lib.workspace_size("mkv_assign_pages_workspace_size", self.rows, self.max_blocks)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        stride = self.block_tables.stride(0) if self.rows > 1 else self.max_blocks
        _call_on(self.device, "mkv_assign_pages", *self.pages._pools, self.block_tables.data_ptr(), stride,
                 self.max_blocks, self.seq_lens.data_ptr(), self.held.data_ptr(), self.ref_counts.data_ptr(),
                 parents.data_ptr(), codes[0], None if tokens is None else tokens.data_ptr(), codes[1],
                 granted.data_ptr(), self.rows, ws.data_ptr(), nbytes, _stream(self.device))
        return granted

    def trim(self) -> None:
        """Let every row go of its pages past those of seq_lens tokens (after an
        eviction has shortened sequences, say).  On the device, in place; pages that
        other rows hold too stay theirs."""
        stride = self.block_tables.stride(0) if self.rows > 1 else self.max_blocks
        _call_on(self.device, "mkv_trim_pages", self.block_tables.data_ptr(), stride, self.max_blocks,
                 self.seq_lens.data_ptr(), self.held.data_ptr(), self.ref_counts.data_ptr(), self.pages.num_blocks,
                 self.pages.block_size, self.rows, _stream(self.device))

    def _parents(self, rows: Sequence[int], parent: int) -> torch.Tensor:
        rows = list(rows)
        if not all(0 <= r < self.rows for r in rows) or len(set(rows)) != len(rows):
            raise ValueError(f"rows must be unlike and in 0..{self.rows - 1}; got {rows}")
        parents = torch.arange(self.rows, dtype=torch.int64)
        parents[rows] = parent
        return parents.to(self.device)

    def fork(self, row: int, rows: Sequence[int]) -> torch.Tensor:
        """Let the given rows go on with row's sequence (see :meth:`assign`)."""
        rows = list(rows)
        if not 0 <= row < self.rows or row in rows:
            raise ValueError(f"row {row} must be one of 0..{self.rows - 1} and not among {rows}")
        return self.assign(self._parents(rows, row))

    def free(self, rows: Sequence[int]) -> None:
        """Free the given rows' sequences (see :meth:`assign`)."""
        self.assign(self._parents(rows, -1))
