"""GPU parity of decode and chunked prefill over 1-byte caches with queries near
zero (every visible key weighs the same), against the oracle."""
from __future__ import annotations

import pytest
import torch

from conftest import announce, assert_close_out
from mkv import attention as A
from oracle import reference as R
from test_gpu_quant import FP8_MODE, INT8_MODE, _prefill_case, _prefill_gpu, _run

pytestmark = pytest.mark.gpu

SIZES = [(torch.bfloat16, 1e-37), (torch.bfloat16, 1e-39), (torch.float32, 1e-37)]


def _case(mode, prior, qlen, Hq, Hkv, qdt, size):
    tensor = mode == "fp8_per_tensor"
    q, kq, vq, ks, vs, bt, ctx, cu, pos = _prefill_case(74, FP8_MODE if tensor else mode, prior, qlen, Hq, Hkv, 16)
    if tensor:
        ks, vs = torch.tensor([0.013]), torch.tensor([0.011])
    q = (q.float() * size).to(qdt)
    assert bool((q != 0).any())
    return q, kq, vq, ks, vs, bt, ctx, cu, pos


def _check(got, q, kq, vq, ks, vs, bt, ctx, cu, pos, Hq, Hkv):
    """P is 1 for every key, exact in fp16, but for per-token V scales folded into
    it (2^-11); the rest are fp32 sums of at most 120 terms."""
    scales = (float(ks), float(vs)) if ks.numel() == 1 else (ks, vs)
    want = R.paged_prefill_ref(q.double(), kq, vq, bt, ctx, cu, pos, 0.1, Hq, Hkv, *scales)
    top = float((vq.float() * (vs if vs.numel() == 1 else vs[..., None])).abs().max())
    assert_close_out(got, want, got.dtype, top * (2.0 ** -11 + 2.0 ** -16))


@pytest.mark.parametrize("mode", ["fp8_per_tensor", FP8_MODE, INT8_MODE])
@pytest.mark.parametrize("qdt,size", SIZES)
def test_prefill(dev, mode, qdt, size):
    announce(f"prefill {mode}, q {qdt} at {size}")
    c = _case(mode, [0, 100], [70, 20], 8, 2, qdt, size)
    q, kq, vq, ks, vs, bt, ctx, cu, pos = c
    _check(_prefill_gpu(dev, mode, q, kq, vq, ks, vs, bt, ctx, cu, pos, 0.1, 8, 2), *c, 8, 2)


@pytest.mark.parametrize("mode", ["fp8_per_tensor", FP8_MODE, INT8_MODE])
@pytest.mark.parametrize("qdt,size", SIZES)
@pytest.mark.parametrize("split", [0, 32, A.DECODE_STREAM, A.DECODE_WORKGROUP])
def test_decode(dev, mode, qdt, size, split):
    announce(f"decode {mode}, q {qdt} at {size}, split {split}")
    c = _case(mode, [69, 119, 0], [1, 1, 1], 8, 2, qdt, size)
    q, kq, vq, ks, vs, bt, ctx, cu, pos = c
    if mode == "fp8_per_tensor":
        got = A.paged_attention_decode_quantized(q.to(dev), kq.to(dev), vq.to(dev), ks.to(dev), vs.to(dev), bt.to(dev),
                                                 ctx.to(dev), 0.1, 8, 2, 128, 16, mode, split_tokens=split).cpu()
    else:
        got = _run(dev, mode, q, kq, vq, ks, vs, bt, ctx, 0.1, 8, 2, split_tokens=split)
    _check(got, *c, 8, 2)
