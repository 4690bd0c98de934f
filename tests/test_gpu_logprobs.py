"""GPU parity of token log probabilities, entropy and top alternatives against
log_softmax in float64.

Bounds.  All arithmetic is fp32: x - m and its exponential each carry 2^-23
relative to the value (the exponential of an argument near -20 a further 20 x
2^-24), sums of up to 32 terms a thread and a tree beyond grow by 40 x 2^-24 at
most, the logarithm adds 2^-23 of at most 18: below 1e-5 for log probabilities
down to -60, taken relative to their size beyond; the entropy sums e (x - m),
|x - m| <= 60 where e is not 0: below 3e-5."""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce
from mkv.decode_state import graph_capture

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def expected(logits, ids, top):
    x = logits.double()
    lp = torch.log_softmax(x, -1)
    bad = ids.clamp(0, x.shape[1] - 1)
    got = lp.gather(1, bad)
    got = torch.where(ids < 0, 0.0, torch.where(ids >= x.shape[1], math.nan, got))
    p = lp.exp()
    entropy = -torch.where((p > 0) | p.isnan(), p * lp, 0.0).sum(-1)
    order = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    return got, entropy, lp.gather(1, order), order


def compare(logits, ids, top, dev, gpu_logits=None):
    """ids (rows, n); logits on the CPU."""
    r = mkv.token_logprobs(logits.to(dev) if gpu_logits is None else gpu_logits, ids.to(dev), top)
    want = expected(logits, ids, top)
    assert torch.equal(r.top_indices.cpu(), want[3])
    for name, got, ref, tol in (("logprobs", r.logprobs, want[0], 1e-5), ("entropy", r.entropy, want[1], 3e-5),
                                ("top", r.top_logprobs, want[2], 1e-5)):
        got = got.double().cpu()
        assert got.shape == ref.shape
        fine = torch.isfinite(ref)
        assert torch.equal(got.isnan(), ref.isnan()), name
        assert torch.equal(got[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()]), name
        err = (got - ref)[fine].abs() - tol * ref[fine].abs().clamp(min=1.0)
        assert err.numel() == 0 or float(err.max()) <= 0, (name, float(err.max()))
    return r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 100, 64), (4, 1003, 20), (2, 8191, 5),
                                            (3, 8192, 64), (2, 8193, 1), (3, 50257, 20), (60, 151936, 5),
                                            (1, 262144, 64), (1, 1000003, 7)])
def test_against_log_softmax(dev, dtype, rows, vocab, top):
    announce(f"logprobs {dtype} {rows}x{vocab} top {top}")
    g = torch.Generator().manual_seed(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    compare(logits, torch.randint(vocab, (rows, 3), generator=g), top, dev)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(dev, dtype):
    announce(f"logprobs ties {dtype}")
    g = torch.Generator().manual_seed(1)
    V = 40000
    rows = [torch.zeros(V), torch.full((V,), -math.inf), torch.randint(0, 3, (V,), generator=g).float(),
            torch.zeros(V), torch.full((V,), -math.inf), torch.arange(V) % 2 - 1.0, torch.zeros(V)]
    rows[3][39990:] = 1.0
    rows[4][[17, 30000, 39999]] = torch.tensor([0.5, 0.5, -2.0])
    rows[6][::3] = -0.0
    logits = torch.stack(rows).to(dtype)
    for top in (1, 5, 64):
        compare(logits, torch.tensor([[0, V - 1]] * len(rows)), top, dev)
    # many near the top in one thread's share (pieces of 8 a chunk apart), and
    # everywhere
    x = torch.randn(3, V, generator=g)
    x[0, :8] = 9.0
    x[0, 2048:2056] = 9.0
    x[1, 100:4000] = 5.0
    x[2, 20000:20100] = torch.linspace(5, 6, 100)
    compare(x.to(dtype), torch.zeros(3, 1, dtype=torch.int64), 64, dev)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_infinite_and_nan_logits(dev, dtype):
    announce(f"logprobs not finite {dtype}")
    g = torch.Generator().manual_seed(2)
    V = 20000
    x = torch.randn(8, V, generator=g) * 2
    x[0, torch.rand(V, generator=g) < 0.9] = -math.inf
    x[1] = -math.inf
    x[1, 12345] = 1.0
    x[2] = -math.inf
    x[3, 77] = math.inf
    x[4, 9000] = math.nan
    x[5] = math.nan
    x[6, 5] = x[6, 15000] = math.inf
    x[6, 8] = math.nan
    x[7] = torch.finfo(dtype).min
    x[7, 3] = 2.0
    ids = torch.tensor([[12345, 3, 77]] * 8)
    compare(x.to(dtype), ids, 20, dev)


def test_far_values(dev):
    """Logits far apart, and far from zero: no overflow, probabilities of 0."""
    announce("logprobs far")
    x = torch.randn(4, 9000)
    x[0] *= 1e4
    x[1] += 3e4
    x[2] = -1e30
    x[2, 5] = 3e38
    x[3] = torch.linspace(-200, 0, 9000)
    r = mkv.token_logprobs(x.to(dev), torch.tensor([1, 2, 5, 0], device=dev), 3)
    want = expected(x, torch.tensor([[1], [2], [5], [0]]), 3)
    assert torch.equal(r.top_indices.cpu(), want[3])
    # (x - m is one fp32 subtraction: 2^-24 of the larger of the two)
    scale = torch.tensor([4e4, 3e4, 1.0, 200.0]).double()
    assert bool(((r.logprobs.double().cpu() - want[0][:, 0]).abs() <= scale * 2e-6 + 1e-5).all())
    assert bool(((r.entropy.double().cpu() - want[1]).abs() <= 3e-5 + 2e-6 * scale).all())


def test_ids_and_layouts(dev):
    announce("logprobs layouts")
    g = torch.Generator().manual_seed(3)
    V = 5003
    logits = torch.randn(6, V, generator=g).to(torch.bfloat16)
    ids = torch.tensor([[0, -1, V], [V - 1, -100, 2], [5, 5, 5], [-1, -1, -1], [1 << 40, 1, 0], [7, 8, V + 1]])
    want = compare(logits, ids, 5, dev)
    # rows at odd places, a column slice, int32 ids with a stride, one id a row
    for off in range(9):
        big = torch.zeros(6, V + 21, dtype=torch.bfloat16, device=dev)
        view = big[:, off:off + V]
        view.copy_(logits)
        # (a row's start decides which logits a thread sums: alike within the
        # bounds, not bit for bit)
        compare(logits, ids, 5, dev, gpu_logits=view)
    r = mkv.token_logprobs(logits.to(dev).t().contiguous().t(), ids[:, 0].to(dev), 0)
    assert r.logprobs.shape == (6,) and r.top_logprobs.shape == (6, 0)
    assert torch.equal(r.logprobs[:3], want.logprobs[:3, 0])  # (copied to the same layout)
    wide = torch.stack([ids.clamp(-1, V), ids.clamp(-1, V)], 2).to(torch.int32).to(dev)
    r = mkv.token_logprobs(logits.to(dev), wide[:, :, 0], 5)
    assert torch.equal(r.logprobs[:4].nan_to_num(9), want.logprobs[:4].nan_to_num(9))
    many = torch.randint(V, (6, 700), generator=g)
    compare(logits, many, 1, dev)
    assert mkv.token_logprobs(logits[:0].to(dev), ids[:0].to(dev), 3).top_indices.shape == (0, 3)
    assert mkv.token_logprobs(logits.to(dev), ids[:, :0].to(dev), 3).logprobs.shape == (6, 0)


def test_more_rows_than_a_grid_dimension(dev):
    announce("logprobs many rows")
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(70000, 5, generator=g)
    compare(logits, torch.randint(5, (70000, 1), generator=g), 2, dev)


def test_captured_and_replayed(dev):
    announce("logprobs graph")
    g = torch.Generator().manual_seed(5)
    sets = [((torch.randn(7, 30000, generator=g) * 4).to(torch.bfloat16).to(dev),
             torch.randint(30000, (7, 2), generator=g).to(dev)) for _ in range(3)]
    want = [mkv.token_logprobs(x, t, 9) for x, t in sets]
    x, t = sets[0][0].clone(), sets[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        r = mkv.token_logprobs(x, t, 9)
    for turn in range(5):
        x.copy_(sets[turn % 3][0])
        t.copy_(sets[turn % 3][1])
        graph.replay()
        mkv.token_logprobs(sets[1][0], sets[1][1], 3)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, want[turn % 3])), turn


def test_on_another_stream(dev):
    announce("logprobs stream")
    g = torch.Generator().manual_seed(6)
    x, t = torch.randn(9, 70000, generator=g).to(dev), torch.randint(70000, (9,), generator=g).to(dev)
    want = mkv.token_logprobs(x, t, 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(mkv.token_logprobs(x, t, 4))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
