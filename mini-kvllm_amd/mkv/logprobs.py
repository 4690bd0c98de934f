"""Log probabilities of given tokens, with entropy and top alternatives.

One pass over the logits (mkv_token_logprobs); used for the tokens that an
engine samples, for scoring a prompt, and for the drafted tokens of a
verification step.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .attention import _call_on, _dtype_code, _require_gpu, _stream

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    """logprobs: fp32, token_ids' shape.  entropy: fp32 (rows,), in nats.
    top_logprobs, top_indices: fp32 and int64 (rows, top), larger first, the
    lower index first among equal logits."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_indices: torch.Tensor


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """log softmax(logits) at token_ids, the entropy of each row's
    distribution, and its ``top`` (0 to 64, at most the vocabulary) likeliest
    tokens.

    logits: fp32, bf16 or fp16 (rows, vocab), rows any stride apart; token_ids:
    int64 or int32 (rows,) or (rows, n).  A negative id marks an absent token (0);
    one past the vocabulary gives NaN.  -inf logits are tokens of probability 0; a
    row with a NaN or +inf, or -inf alone, has NaN log probabilities.  The
    arithmetic is fp32; nothing is recorded for gradients."""
    dev = _require_gpu(logits, token_ids)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be (rows, vocab); got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits: unsupported dtype {logits.dtype}")
    if token_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token_ids must be int32 or int64, got {token_ids.dtype}")
    if token_ids.dim() not in (1, 2) or token_ids.shape[0] != rows:
        raise ValueError(f"token_ids must be ({rows},) or ({rows}, n); got {tuple(token_ids.shape)}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top {top} outside 0..{min(MAX_TOP, vocab)}")
    if logits.stride(1) != 1 or logits.stride(0) < vocab:
        logits = logits.contiguous()
    ids = token_ids if token_ids.dim() == 2 else token_ids[:, None]
    if ids.shape[1] and (ids.stride(1) != 1 or ids.stride(0) < ids.shape[1]):
        ids = ids.contiguous()
    num_ids = ids.shape[1]
    out = TokenLogprobs(torch.empty(token_ids.shape, dtype=torch.float32, device=dev),
                        torch.empty(rows, dtype=torch.float32, device=dev),
                        torch.empty(rows, top, dtype=torch.float32, device=dev),
                        torch.empty(rows, top, dtype=torch.int64, device=dev))
    if rows == 0:
        return out
    nbytes = _lib.workspace_size("mkv_token_logprobs_workspace_size", rows, vocab, top)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call_on(dev, "mkv_token_logprobs", out.logprobs.data_ptr(), out.entropy.data_ptr(),
             out.top_logprobs.data_ptr(), out.top_indices.data_ptr(), logits.data_ptr(),
             # (the stride of a single row means nothing)
             logits.stride(0) if rows > 1 else vocab, _dtype_code(logits, "logits"), rows, vocab, ids.data_ptr(),
             ids.stride(0) if rows > 1 else num_ids, num_ids,
             _lib.INDEX_I64 if ids.dtype == torch.int64 else _lib.INDEX_I32, top, ws.data_ptr(), nbytes, _stream(dev))
    return out
