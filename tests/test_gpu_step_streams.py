"""GPU tests of the speculative step's operators in the settings they are used
in: batches past 64 sequences and rows in many splits, streams of their own,
captured graphs."""
from __future__ import annotations

import pytest
import torch

import mkv
from conftest import announce
from mkv.decode_state import graph_capture
from test_gpu_pages import MIXES, caches, same
from test_gpu_tree import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8", "int8_token"])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (16, 2)])
def test_more_sequences_than_a_wave_has_lanes(dev, fmt, heads, kv_heads):
    """Short sequences with a few long ones, on both sides of the 64th and the
    128th: the long ones are split, and their places are counted past 64."""
    announce(f"tree, 150 sequences, {fmt}, {heads} heads over {kv_heads}")
    drafted = [1 + (7 * i) % 6 for i in range(150)]
    prefix = [(11 * i) % 50 for i in range(150)]
    for i, p in ((3, 2500), (63, 1800), (64, 4100), (100, 3000), (149, 2600)):
        prefix[i] = p
    drafted[70] = drafted[127] = 0
    check(make(fmt, drafted, prefix, heads, kv_heads, 128, 16, seed=2), dev)


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8"])
@pytest.mark.parametrize("drafted,prefix,heads", [([6], [9000], 2), ([40], [5000], 2), ([64, 50], [6000, 7000], 4),
                                                  ([64] * 9, [1500] * 9, 8)])
def test_rows_in_many_splits(dev, fmt, drafted, prefix, heads):
    announce(f"tree, splits, {fmt}, {drafted[0]} of {prefix[0]}")
    c = make(fmt, drafted, prefix, heads, 1, 128, 16, seed=5)
    got = check(c, dev)
    assert torch.equal(got, run(c, dev, ctx=c["ctx"].to(torch.int32), cu=c["cu"].to(torch.int64)))


def test_streams_of_their_own(dev):
    """Every operator on a side stream, ahead of which its inputs are made
    there: the default stream is kept busy with other work meanwhile."""
    announce("step operators on a side stream")
    c = make("bf16", [9, 3], [700, 90], 8, 2, 128, 16, seed=3)
    want = run(c, dev)
    ts = caches(dev, 12, 16, MIXES["bf16"], seed=4)
    copied = [t.clone() for t in ts]
    for w in copied:
        w[[5, 6]] = w[[1, 2]]
        w[1, 3:5] = w[1, [4, 7]]
    logits = torch.randn(7, 9000, device=dev)
    lp = mkv.token_logprobs(logits, torch.arange(7, device=dev), 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(dev)
    busy = torch.randn(2048, 2048, device=dev)
    for _ in range(20):
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(side):
        got = run(c, dev)
        fresh = logits.clone()
        r = mkv.token_logprobs(fresh, torch.arange(7, device=dev), 4)
        pages = mkv.CachePages(ts)
        pages.copy([1, 2], [5, 6])
        pages.compact(torch.tensor([[1]], dtype=torch.int32, device=dev), torch.tensor([3], device=dev),
                      torch.tensor([[1, 4]], device=dev))
    side.synchronize()
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(r, lp))
    assert all(same(a, b) for a, b in zip(ts, copied))


def test_copy_and_compact_captured_and_replayed(dev):
    """One graph of a page copy and a compaction over fixed buffers whose
    contents change between replays, with eager calls beside them."""
    announce("copy and compact graph")
    ts = caches(dev, 16, 16, MIXES["token"], seed=6)
    start = [t.clone() for t in ts]
    pages = mkv.CachePages(ts)
    src, dst = (torch.tensor(x, device=dev) for x in ([0, 1], [8, 9]))
    bt = torch.tensor([[0, 1, -1], [2, 3, 4]], dtype=torch.int32, device=dev)
    prefix, accepted = torch.tensor([14, 30], device=dev), torch.tensor([[0, 2, 5], [3, 4, -1]], device=dev)

    def step():
        pages.copy(src, dst)
        pages.compact(bt, prefix, accepted)

    step()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        step()
    plans = [([0, 1], [8, 9], [14, 30], [[0, 2, 5], [3, 4, -1]]), ([5, 0], [6, 7], [3, 17], [[1, 2, 9], [0, 1, 2]]),
             ([2, 4], [12, 15], [0, 31], [[4, 8, 12], [1, 2, 3]])]
    for turn in range(6):
        s, d, p, acc = plans[turn % 3]
        for t, x in ((src, s), (dst, d), (prefix, p), (accepted, acc)):
            t.copy_(torch.tensor(x))
        want = []
        for t, x in zip(ts, start):
            t.copy_(x)
            w = x.clone()
            w[d] = w[s]
            flat = w.view(16 * 16, *w.shape[2:])
            for row in range(2):
                def at(pos):
                    return int(bt[row, pos // 16]) * 16 + pos % 16
                moves = [(at(p[row] + a), at(p[row] + j)) for j, a in enumerate(acc[row]) if a >= 0]
                moved = [flat[a].clone() for a, _ in moves]
                for (_, b), v in zip(moves, moved):
                    flat[b] = v
            want.append(w)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(ts, want)), f"replay {turn}"
        for t, x in zip(ts, start):  # eager work between the replays
            t.copy_(x)
        step()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(ts, want)), f"eager {turn}"
