"""Verification of drafted tokens against the target model's distribution.

The accepting half of speculative sampling (mkv_verify_drafts): it takes the
logits that a step with drafted tokens ends with (a chain's or a tree's, see
:func:`mkv.paged_attention_tree`) and says which of them stay, for
:meth:`mkv.CachePages.compact`, and what comes next.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .attention import _call_on, _dtype_code, _require_gpu, _stream

MAX_NODES = 1024


class VerifiedDrafts(NamedTuple):
    """accepted: int64 (seqs, max_nodes), each sequence's path through its nodes
    (node 0 first), -1 behind it: the offsets that CachePages.compact takes.
    num_accepted: int64 (seqs,), the path's length.  next_tokens: int64 (seqs,).
    acceptance: fp32 (total,), each node's chance of being accepted as the first
    of its siblings."""

    accepted: torch.Tensor
    num_accepted: torch.Tensor
    next_tokens: torch.Tensor
    acceptance: torch.Tensor


def verify_drafts(logits: torch.Tensor, token_ids: torch.Tensor, cu_seqlens_q: torch.Tensor,
                  uniforms: torch.Tensor, noise: torch.Tensor, max_nodes: int, *,
                  parents: torch.Tensor | None = None, draft_logits: torch.Tensor | None = None,
                  temperatures: torch.Tensor | None = None) -> VerifiedDrafts:
    """Accept drafted tokens so that what is generated follows the target's
    distribution, and draw the token behind them.

    logits: fp32, bf16 or fp16 (total, vocab), the target's behind every node, the
    nodes of every sequence one after another (cu_seqlens_q, int32 (seqs + 1,)).
    Node 0 of a sequence is its last token, the others are drafted: token_ids
    (total,), and parents (total,), offsets within the sequence below the node's own
    (node 0's is not looked at; None: chains).  draft_logits: logits' shape and type,
    the draft's behind each node, from which its children's tokens were drawn one by
    one (rows without children are not read); None: the tokens were picked without
    drawing (likeliest tokens, copied text).  temperatures: fp32 (seqs,), of target and
    draft; 0 is greedy.

    From uniforms (fp32 (total,), in [0, 1)) a child x of the node reached, in the
    order of its siblings, is accepted if u q(x) < p(x); else p becomes max(0, p - q),
    normalised.  The next token is argmax p / noise of what is left behind the last
    node accepted, noise (fp32 (seqs, vocab)) being Exp(1) variates: the engine's own
    way of sampling.  Ties go to the lowest index.

    max_nodes (up to 1024): the most nodes of a sequence; those past it are not looked
    at.  Rows of acceptance that are no sequence's are not written.  A row with a NaN
    or +inf, or -inf alone, is taken as greedy; tokens outside the vocabulary and nodes
    whose parent is no earlier node are never accepted."""
    dev = _require_gpu(logits, token_ids, cu_seqlens_q, uniforms, noise,
                       *(t for t in (parents, draft_logits, temperatures) if t is not None))
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be (total, vocab); got {tuple(logits.shape)}")
    total, vocab = logits.shape
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits: unsupported dtype {logits.dtype}")
    if draft_logits is not None and (draft_logits.shape != logits.shape or draft_logits.dtype != logits.dtype):
        raise ValueError(f"draft_logits must be a {logits.dtype} tensor of {tuple(logits.shape)}; got "
                         f"{draft_logits.dtype} {tuple(draft_logits.shape)}")
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.numel() == 0:
        raise ValueError(f"cu_seqlens_q must be (seqs + 1,); got {tuple(cu_seqlens_q.shape)}")
    num_seqs = cu_seqlens_q.numel() - 1
    if num_seqs > 65535:
        raise ValueError(f"{num_seqs} sequences > 65535")
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes {max_nodes} outside 1..{MAX_NODES}")
    for name, t in (("token_ids", token_ids), ("parents", parents)):
        if t is not None and (t.shape != (total,) or t.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"{name} must be int32 or int64 ({total},); got {t.dtype} {tuple(t.shape)}")
    for name, t, shape in (("uniforms", uniforms, (total,)), ("noise", noise, (num_seqs, vocab)),
                           ("temperatures", temperatures, (num_seqs,))):
        if t is not None and (t.shape != shape or t.dtype != torch.float32):
            raise ValueError(f"{name} must be float32 {shape}; got {t.dtype} {tuple(t.shape)}")

    def rows(t):
        return t if t.stride(1) == 1 and t.stride(0) >= vocab else t.contiguous()

    def code(t):
        return _lib.INDEX_I64 if t.dtype == torch.int64 else _lib.INDEX_I32

    logits, noise = rows(logits), rows(noise)
    draft_logits = None if draft_logits is None else rows(draft_logits)
    token_ids, uniforms = token_ids.contiguous(), uniforms.contiguous()
    parents = None if parents is None else parents.contiguous()
    temperatures = None if temperatures is None else temperatures.contiguous()
    cu = cu_seqlens_q.to(torch.int32).contiguous()
    out = VerifiedDrafts(torch.empty(num_seqs, max_nodes, dtype=torch.int64, device=dev),
                         torch.empty(num_seqs, dtype=torch.int64, device=dev),
                         torch.empty(num_seqs, dtype=torch.int64, device=dev),
                         torch.empty(total, dtype=torch.float32, device=dev))
    if num_seqs == 0:
        return out
    nbytes = _lib.workspace_size("mkv_verify_drafts_workspace_size", total, vocab, num_seqs, max_nodes,
                                 int(draft_logits is not None))
    # (of the call's own: calls on several streams and captured graphs share none)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)

    def ptr(t):
        return None if t is None else t.data_ptr()

    _call_on(dev, "mkv_verify_drafts", *(t.data_ptr() for t in out), logits.data_ptr(),
             # (the stride of a single row means nothing)
             logits.stride(0) if total > 1 else vocab, ptr(draft_logits),
             draft_logits.stride(0) if draft_logits is not None and total > 1 else vocab, _dtype_code(logits, "logits"),
             total, vocab, token_ids.data_ptr(), code(token_ids), ptr(parents), 0 if parents is None else code(parents),
             cu.data_ptr(), num_seqs, max_nodes, uniforms.data_ptr(), noise.data_ptr(),
             noise.stride(0) if num_seqs > 1 else vocab, ptr(temperatures), ws.data_ptr(), nbytes, _stream(dev))
    return out
