"""Eviction from the KV cache by accumulated attention weight.

:func:`mkv.paged_attention_weights` keeps, beside every layer's cache, the weight
that each cached token has received; :class:`CacheEviction` shortens sequences to a
budget by it, every layer and KV head for itself, and :meth:`mkv.PagePool.trim`
gives back the pages that this frees.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from . import _lib
from .attention import _block_table, _call_on, _require_gpu, _stream
from .pages import _index_code

MAX_HEAD_BYTES = 2048


class CacheEviction:
    """All layers' K and V pools (num_blocks, block_size, num_kv_heads, head_dim),
    their accumulated weights, fp32 (num_blocks, block_size, num_kv_heads), and, with
    per-token-head formats, their scales of that shape: contiguous, none overlapping
    another.  The tensors are kept; they must stay where they are.  ``tensors``: all of
    them, what :class:`mkv.CachePages` takes so that page copies and compactions bring
    a token's weights along."""

    def __init__(self, k_caches: Sequence[torch.Tensor], v_caches: Sequence[torch.Tensor],
                 weights: Sequence[torch.Tensor], k_scales: Sequence[torch.Tensor] | None = None,
                 v_scales: Sequence[torch.Tensor] | None = None):
        groups = [list(k_caches), list(v_caches), list(weights)]
        if (k_scales is None) != (v_scales is None):
            raise ValueError("k_scales and v_scales go together")
        if k_scales is not None:
            groups += [list(k_scales), list(v_scales)]
        self.num_layers = len(groups[0])
        if not self.num_layers or any(len(x) != self.num_layers for x in groups):
            raise ValueError(f"every layer needs each of its tensors; got {[len(x) for x in groups]}")
        self.tensors = [t for x in groups for t in x]
        # tables whose sequences' lengths and positions are the host's (mkv.engine.Engine)
        self.engine_tables: torch.Tensor | None = None
        self.device = _require_gpu(*self.tensors)
        shape = groups[0][0].shape
        if len(shape) != 4 or not all(shape):
            raise ValueError(f"a cache must be (num_blocks, block_size, num_kv_heads, head_dim); got {tuple(shape)}")
        self.num_blocks, self.block_size, self.num_kv_heads = shape[:3]
        if self.block_size < 4 or self.block_size & (self.block_size - 1):
            raise ValueError(f"block_size must be a power of two from 4 on; got {self.block_size}")
        if self.num_kv_heads > 1024 or self.num_blocks * self.block_size > 0x7fffffff:
            raise ValueError(f"a cache of {tuple(shape)} has too many heads or tokens")
        rows = self.num_blocks * self.block_size * self.num_kv_heads
        sizes = []
        for i, t in enumerate(self.tensors):
            if i < 2 * self.num_layers:
                if t.dim() != 4 or t.shape[:3] != shape[:3]:
                    raise ValueError(f"caches of {tuple(t.shape)} and {tuple(shape)}")
            elif t.shape != shape[:3] or t.dtype != torch.float32:
                raise ValueError(f"weights and scales must be float32 {tuple(shape[:3])}; got {t.dtype} {tuple(t.shape)}")
            if not t.is_contiguous():
                raise ValueError("cache tensors must be contiguous")
            size = t.nbytes // rows
            if size == 0 or size % 4 or size > MAX_HEAD_BYTES or t.data_ptr() % 4:
                raise ValueError(f"a head's row must be a multiple of 4 bytes up to {MAX_HEAD_BYTES}; got "
                                 f"{tuple(t.shape)} {t.dtype}")
            sizes.append(size)
        ptrs = [t.data_ptr() for t in self.tensors]
        spans = sorted(zip(ptrs, sizes))
        if any(a + n * rows > b for (a, n), (b, _) in zip(spans, spans[1:])):
            raise ValueError("cache tensors overlap")
        n, L = len(ptrs), self.num_layers
        self._ptrs, self._sizes = (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*sizes)
        self._layers = (ctypes.c_int * n)(*(i % L for i in range(n)))
        self._weights = (ctypes.c_void_p * L)(*ptrs[2 * L:3 * L])
        self._args = (ctypes.addressof(self._ptrs), ctypes.addressof(self._sizes), ctypes.addressof(self._layers), n,
                      ctypes.addressof(self._weights), L, self.num_blocks, self.block_size, self.num_kv_heads)

    def evict(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, budget: int, *, sinks: int = 0,
              recent: int = 0) -> torch.Tensor:
        """Cut every sequence of more than ``budget`` tokens to that many, in every
        layer and KV head: the first ``sinks`` and the last ``recent`` (together at
        most the budget) stay, and of the others those of the largest weight (the
        earlier of equal ones; NaN is larger than all).  What stays moves to positions
        0 .. budget - 1 in its order, each head's rows of K, V, weights and scales for
        itself; what lies behind is left as it was.

        block_tables: int32 (batch or more, blocks); seq_lens: int32 or int64 (batch,),
        the tokens in the cache.  Returns the new lengths, int64 (batch,), min(length,
        budget), the context_lens of what follows; the positions that tokens had (their
        rotary angles) go on from the old lengths.  On the device, without a word from
        the host.  Sequences must not share pages of the positions below the budget
        (forks: evict first); the tables' pages must be in the pool."""
        _require_gpu(self.tensors[0], block_tables, seq_lens)
        if (self.engine_tables is not None
                and block_tables.untyped_storage().data_ptr() == self.engine_tables.untyped_storage().data_ptr()):
            raise ValueError("these are an Engine's sequences: it goes by its host's lengths and positions, which a cut "
                             "does not change")
        if seq_lens.dim() != 1 or block_tables.dim() != 2 or block_tables.shape[0] < seq_lens.numel():
            raise ValueError(f"block_tables {tuple(block_tables.shape)} must cover seq_lens {tuple(seq_lens.shape)}")
        if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError(f"budget {budget} must be at least 1 and hold {sinks} sinks and {recent} recent tokens")
        batch = seq_lens.numel()
        if batch > 65535:
            raise ValueError(f"batch {batch} > 65535")
        code = _index_code(seq_lens, "seq_lens")
        bt, seq_lens = _block_table(block_tables), seq_lens.contiguous()
        if batch == 0 or bt.shape[1] * self.block_size <= budget:  # (no table holds more)
            return seq_lens.to(torch.int64).clamp(0, budget)
        new = torch.empty(batch, dtype=torch.int64, device=self.device)
        nbytes = _lib.workspace_size("mkv_evict_tokens_workspace_size", self.num_layers, batch, self.num_kv_heads,
                                     self.block_size, bt.shape[1], budget)
        # (of the call's own: calls on several streams and captured graphs share none)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        _call_on(self.device, "mkv_evict_tokens", *self._args, bt.data_ptr(), bt.stride(0) if batch > 1 else bt.shape[1],
                 bt.shape[1], seq_lens.data_ptr(), code, batch, budget, sinks, recent, new.data_ptr(), ws.data_ptr(),
                 nbytes, _stream(self.device))
        return new
