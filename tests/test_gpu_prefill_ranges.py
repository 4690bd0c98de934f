"""GPU parity of the chunked prefill over per-token-head caches with V scales of any
size, against the oracle."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import announce
from oracle import reference as R
from test_gpu_quant import FP8_MODE, INT8_MODE, _prefill_case, _prefill_gpu

pytestmark = pytest.mark.gpu


def _close(got, q, kq, vq, ks, vs, bt, ctx, cu, pos, sc, Hq, Hkv, keys):
    """Each output by itself.  With A = sum p |v| / sum p: P times the V scale is
    rounded to fp16 once (2^-11 A); the fp32 arithmetic's parts are relative to the
    terms (2^-11 A, as for tree attention); products below fp16's normal range are
    off by up to 2^-25 where the largest P times its tile's largest V scale is 2^6
    or more (2^-31 of the largest |v| a key); the store's half step."""
    args = bt, ctx, cu, pos, sc, Hq, Hkv
    want = R.paged_prefill_ref(q.double(), kq, vq, *args, ks, vs)
    a = R.paged_prefill_ref(q.double(), kq, vq.float().abs(), *args, ks, vs)
    tol = 2.0 ** -10 * a + keys * 2.0 ** -31 * float((vq.float() * vs[..., None]).abs().max())
    if q.dtype == torch.bfloat16:
        tol = tol + torch.where(want == 0, 0.0, 0.5 * torch.exp2(torch.floor(torch.log2(want.abs())) - 7))
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (f"{int((~(err <= tol)).sum())} of {err.numel()} out of tolerance; largest error "
                                      f"{float(err.nan_to_num(math.inf).max()):.3e}")


@pytest.mark.parametrize("mode", [FP8_MODE, INT8_MODE])
@pytest.mark.parametrize("qdt,group", [(torch.bfloat16, 4), (torch.float32, 4), (torch.bfloat16, 16)])
@pytest.mark.parametrize("power", [-38, -20, -10, 20])
def test_v_scales_of_any_size(dev, mode, qdt, group, power):
    """V scales 2^power times the usual: that times the output (exactly, a power
    of two), within the bound of the usual ones."""
    announce(f"per-token prefill {mode} q {qdt} group {group}, V scales x 2^{power}")
    Hkv = 2
    case = _prefill_case(60 + group, mode, [0, 400, 90], [130, 70, 200], Hkv * group, Hkv, 16, qdt)
    q, kq, vq, ks, vs, bt, ctx, cu, pos = case
    sc = 1 / math.sqrt(128)
    got = _prefill_gpu(dev, mode, q, kq, vq, ks, vs * 2.0 ** power, bt, ctx, cu, pos, sc, Hkv * group, Hkv)
    _close(got.double() / 2.0 ** power, *case, sc, Hkv * group, Hkv, 470)


@pytest.mark.parametrize("mode", [FP8_MODE, INT8_MODE])
@pytest.mark.parametrize("small", [1e-2, 1e-5, 0.0])
def test_a_sink(dev, mode, small):
    """The first token draws most of every row's weight (a logit of 9 above the
    others), and its own V scale is a hundredth, 10^-5 or none of the others'."""
    announce(f"per-token prefill {mode}, a sink with V scale x {small}")
    Hq, Hkv = 8, 2
    q, kq, vq, ks, vs, bt, ctx, cu, pos = _prefill_case(71, mode, [0, 1900], [130, 70], Hq, Hkv, 16)
    ks *= 0.25
    u = torch.where(torch.arange(128) % 3 == 0, -1.0, 1.0)
    for s in range(2):
        page = int(bt[s, 0])
        kq[page, 0] = (u * 16).to(kq.dtype)
        ks[page, 0] = 1 / 32
        vs[page, 0] *= small
    sc = 1 / math.sqrt(128)
    q = (q.float() * 0.2 + 9 / (64 * sc) * u).to(q.dtype)
    got = _prefill_gpu(dev, mode, q, kq, vq, ks, vs, bt, ctx, cu, pos, sc, Hq, Hkv)
    _close(got, q, kq, vq, ks, vs, bt, ctx, cu, pos, sc, Hq, Hkv, 1970)


@pytest.mark.parametrize("mode", [FP8_MODE, INT8_MODE])
def test_no_v_scale_at_all(dev, mode):
    announce(f"per-token prefill {mode}, V scales of 0")
    Hq, Hkv = 8, 2
    q, kq, vq, ks, vs, bt, ctx, cu, pos = _prefill_case(72, mode, [0, 200], [70, 20], Hq, Hkv, 16)
    vs[:] = 0
    got = _prefill_gpu(dev, mode, q, kq, vq, ks, vs, bt, ctx, cu, pos, 0.1, Hq, Hkv)
    assert not bool(got.any())
    # whole tiles without one beside ordinary ones
    q, kq, vq, ks, vs, bt, ctx, cu, pos = _prefill_case(73, mode, [0, 300], [70, 20], Hq, Hkv, 16)
    for s in range(2):
        for j in range(0, 4 if s else 2):
            vs[int(bt[s, j])] = 0
    got = _prefill_gpu(dev, mode, q, kq, vq, ks, vs, bt, ctx, cu, pos, 0.1, Hq, Hkv)
    _close(got, q, kq, vq, ks, vs, bt, ctx, cu, pos, 0.1, Hq, Hkv, 320)
