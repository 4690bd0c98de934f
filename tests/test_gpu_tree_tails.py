"""GPU parity of tree attention over long tails of small weights, which fp16 P has
to hold beside a large one, against its definition."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import announce, assert_close_out
from test_gpu_tree import CACHES, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "fp16", "fp32", "fp8", "fp8_token", "int8_token"])
@pytest.mark.parametrize("bits", [15.0, 25.5])
@pytest.mark.parametrize("seqs,rows", [(1, 1), (64, 128)])
def test_many_small_weights_beside_a_large_one(dev, fmt, bits, seqs, rows):
    """One key of 2^bits times the weight of each of 130,000 others, which
    together weigh up to 4: their V is 1 in every dim and the one's is 0, so the
    output is their share.  One short row, whose keys are spread over many waves,
    and a batch (of one table) where a wave takes whole contexts.  Exactly known:
    q . k is 0 for the others and one product for the one.  fp16 P is off by half a
    step, 2^-11 of it, or by 2^-25 where it is below fp16's normal range and the
    row's largest is 2^7 or more: 2^-32 of the largest weight a key.  The sums are
    fp32, 16 like terms of a lane's block of keys and then the blocks: 130,000 / 32
    additions, half a step each, at 2^-24: 2^-12 of the share; and so are the
    normaliser's."""
    announce(f"tree {fmt}, {seqs} contexts of 130,000 keys of 2^-{bits} of one's weight")
    N, bs, H, D = 130000, 256, 8 if seqs > 1 else 1, 128
    cdt, qdt, mode = CACHES[fmt]
    pages = -(-N // bs) + 2
    k, v = torch.zeros(pages, bs, H, D, device=dev), torch.ones(pages, bs, H, D, device=dev)
    k[1, 3, :, 0], v[1, 3] = 1, 0
    q = torch.zeros(seqs * rows, H, D)
    q[..., 0] = 1
    ks = vs = None
    if mode != "auto":
        ks, vs = (torch.ones(1 if mode == "fp8_per_tensor" else (pages, bs, H)) for _ in range(2))
    bt = (torch.arange(pages - 2, dtype=torch.int32) + 1)[None].expand(seqs, -1).contiguous()
    c = dict(q=q.to(qdt), k=k.to(cdt), v=v.to(cdt), bt=bt, ctx=torch.full((seqs,), N), ks=ks, vs=vs, mode=mode, Hq=H,
             Hkv=H, D=D, bs=bs, cu=torch.arange(seqs + 1, dtype=torch.int32) * rows,
             mask=torch.ones(seqs * rows, rows, dtype=torch.bool), scale=bits * math.log(2))
    got = run(c, dev)
    largest, share = 2.0 ** bits / (2.0 ** bits + N - 1), (N - 1) / (2.0 ** bits + N - 1)
    tol = share * (2.0 ** -11 + 2 * 2.0 ** -12) + N * 2.0 ** -32 * largest
    assert_close_out(got, torch.full(got.shape, share, dtype=torch.float64), got.dtype, tol)
