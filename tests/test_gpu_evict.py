"""GPU tests of the eviction by accumulated attention weight (mkv_evict_tokens)
and of the page table's trim (mkv_trim_pages).  Every result is exact: rows move
as bytes, and the choice is of whole numbers (a stable sort of the weights)."""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce
from mkv import workloads as W
from mkv.decode_state import graph_capture

pytestmark = pytest.mark.gpu


def make(lens, layers, H, D, bs, dtype=torch.bfloat16, scales=False, seed=0, width=None, spare=3):
    """Tensors of every layer on the CPU, and the page tables."""
    g = torch.Generator().manual_seed(seed)
    ctx = torch.tensor(lens, dtype=torch.int64)
    blocks = sum(-(-n // bs) for n in lens) + spare
    bt = W.fragmented_block_tables(ctx, bs, blocks, g)
    if width is not None:
        bt = torch.cat([bt, torch.full((len(lens), max(0, width - bt.shape[1])), -1, dtype=torch.int32)], 1)

    def cache():
        x = torch.randint(0, 256, (blocks, bs, H, D * torch.empty(0, dtype=dtype).element_size()), generator=g)
        return x.to(torch.uint8).view(dtype)

    def row():
        return torch.rand(blocks, bs, H, generator=g)

    c = dict(k=[cache() for _ in range(layers)], v=[cache() for _ in range(layers)], w=[row() for _ in range(layers)])
    if scales:
        c.update(ks=[row() for _ in range(layers)], vs=[row() for _ in range(layers)])
    return c, bt, ctx


def handle(c):
    return mkv.CacheEviction(c["k"], c["v"], c["w"], c.get("ks"), c.get("vs"))


def on(dev, c):
    return {n: [x.to(dev) for x in xs] for n, xs in c.items()}


def oracle(c, bt, lens, budget, sinks, recent):
    """In place, on the CPU."""
    bs, H = c["w"][0].shape[1:]
    for b, n in enumerate(lens.tolist()):
        n = min(n, bt.shape[1] * bs)
        if n <= budget:
            continue
        t = torch.arange(n)
        slots = bt[b, t // bs].long() * bs + t % bs
        for i in range(len(c["w"])):
            w = c["w"][i].flatten(0, 1)[slots].double()
            w = torch.where(torch.isnan(w), math.inf, w)
            # (NaN above +inf: a second key)
            nan = torch.isnan(c["w"][i].flatten(0, 1)[slots]).double()
            for h in range(H):
                mid = sorted(range(sinks, n - recent), key=lambda j: (-float(nan[j, h]), -float(w[j, h]), j))
                keep = list(range(sinks)) + sorted(mid[:budget - sinks - recent]) + list(range(n - recent, n))
                for xs in c.values():
                    x = xs[i].flatten(0, 1)
                    x[slots[:budget], h] = x[slots[keep], h].clone()
    return lens.clamp(0, budget)


def same(got, want):
    for n in want:
        for i, (a, b) in enumerate(zip(got[n], want[n])):
            assert torch.equal(a.cpu().contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), f"{n} of layer {i}"


@pytest.mark.parametrize("dtype,scales", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, True),
                                          (torch.float8_e4m3fn, False), (torch.float8_e4m3fn, True), (torch.int8, True)])
@pytest.mark.parametrize("H,D,bs", [(1, 128, 16), (8, 128, 256), (3, 64, 32), (2, 20, 16)])
def test_sequences_are_cut(dev, dtype, scales, H, D, bs):
    announce(f"evict: {dtype}, scales {scales}, {H} heads of {D}, blocks of {bs}")
    lens = [0, 1, 40, 41, 42, 300, 777, 64]
    c, bt, ctx = make(lens, 2, H, D, bs, dtype, scales, seed=H + D)
    for budget, sinks, recent in ((41, 4, 8), (1, 0, 0), (40, 0, 40), (64, 64, 0), (300, 3, 100)):
        d = on(dev, c)
        want = {n: [x.clone() for x in xs] for n, xs in c.items()}
        lens_want = oracle(want, bt, ctx, budget, sinks, recent)
        new = handle(d).evict(bt.to(dev), ctx.to(dev), budget, sinks=sinks, recent=recent)
        assert new.dtype == torch.int64 and new.tolist() == lens_want.tolist()
        same(d, want)


@pytest.mark.parametrize("width", [None, 600])
def test_equal_and_odd_weights(dev, width):
    """Ties, none but ties, NaN, infinities, negative weights and both zeros; a
    table wider than LDS takes the other way."""
    announce(f"evict: odd weights, table width {width}")
    lens = [700, 90, 333, 512, 65]
    c, bt, ctx = make(lens, 3, 4, 32, 16, seed=3, width=width)
    g = torch.Generator().manual_seed(5)
    c["w"][0] = torch.randint(0, 4, c["w"][0].shape, generator=g).float() / 4
    c["w"][1].zero_()
    odd = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.5, 1e-42, -1e-42, 3.4e38, 2.0])
    c["w"][2] = odd[torch.randint(0, len(odd), c["w"][2].shape, generator=g)]
    c["w"][2][..., 1] = -c["w"][2][..., 1]
    for budget, sinks, recent in ((64, 2, 5), (300, 0, 0), (512, 10, 500)):
        d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
        lens_want = oracle(want, bt, ctx, budget, sinks, recent)
        new = handle(d).evict(bt.to(dev), ctx.to(dev), budget, sinks=sinks, recent=recent)
        assert new.tolist() == lens_want.tolist()
        same(d, want)


def test_long_tables_and_many_layers(dev):
    announce("evict: 20000 tokens; 30 layers; a narrow table")
    c, bt, ctx = make([20000, 150, 9000], 2, 2, 16, 32, seed=6)
    for budget, sinks, recent in ((2500, 4, 64), (9001, 0, 3)):
        d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
        lens_want = oracle(want, bt, ctx, budget, sinks, recent)
        new = handle(d).evict(bt.to(dev), ctx.int().to(dev), budget, sinks=sinks, recent=recent)
        assert new.tolist() == lens_want.tolist()
        same(d, want)
    c, bt, ctx = make([50, 33], 30, 2, 8, 16, scales=True, seed=7)
    d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
    oracle(want, bt, ctx, 20, 1, 2)
    handle(d).evict(bt.to(dev), ctx.to(dev), 20, sinks=1, recent=2)
    same(d, want)
    # lengths past the table: what it holds is cut, the length given is not believed
    c, bt, ctx = make([64, 64], 1, 2, 8, 16, seed=8)
    d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
    oracle(want, bt[:, :3], ctx, 20, 1, 2)
    long = torch.tensor([2 ** 40, -7])
    want["k"], want["v"], want["w"] = want["k"], want["v"], want["w"]
    one = {n: [x.clone() for x in xs] for n, xs in c.items()}
    oracle(one, bt[:1, :3], ctx[:1], 20, 1, 2)
    assert handle(d).evict(bt.to(dev)[:, :3], long.to(dev), 20, sinks=1, recent=2).tolist() == [20, 0]
    same(d, one)
    # a budget that no table reaches: nothing to do
    d = on(dev, c)
    assert handle(d).evict(bt.to(dev), ctx.to(dev), 64).tolist() == [64, 64]
    same(d, c)


def test_rows_longer_than_the_registers_hold(dev):
    """Past 65536 tokens the rest of a row's keys are read again and again; lengths
    that end within a vector of 256, in the table's last page."""
    announce("evict: 66500 and 131073 tokens")
    c, bt, ctx = make([66500, 131073], 1, 2, 4, 16, seed=9)
    for budget, sinks, recent in ((1200, 4, 64), (66400, 0, 1)):
        d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
        oracle(want, bt, ctx, budget, sinks, recent)
        assert handle(d).evict(bt.to(dev), ctx.to(dev), budget, sinks=sinks, recent=recent).tolist() == [budget] * 2
        same(d, want)


@pytest.mark.parametrize("tokens", [1 << 22, 1 << 24])
def test_tables_whose_keys_go_in_turns(dev, tokens):
    """Tables so wide that the room for keys holds some of the layers, or some of a
    layer's sequences, at a time."""
    announce(f"evict: three layers of three sequences under tables of {tokens} tokens")
    c, bt, ctx = make([300, 9000, 77], 3, 2, 8, 16, scales=True, seed=13, width=tokens // 16)
    for budget, sinks, recent in ((60, 2, 5), (301, 0, 20)):
        d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
        lens_want = oracle(want, bt, ctx, budget, sinks, recent)
        new = handle(d).evict(bt.to(dev), ctx.to(dev), budget, sinks=sinks, recent=recent)
        assert new.tolist() == lens_want.tolist()
        same(d, want)


def test_absent_pages_are_left_out(dev):
    """An entry outside the pool: its tokens' weights count as lowest, and no row
    is read from there or written there."""
    announce("evict: absent pages")
    c, bt, ctx = make([100], 1, 2, 8, 16, seed=9)
    bt[0, 2], bt[0, 5] = -1, 10 ** 6
    d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
    t = torch.arange(100)
    here = [int(bt[0, j // 16]) * 16 + j % 16 if j // 16 not in (2, 5) else -1 for j in t.tolist()]
    for h in range(2):
        w = c["w"][0].flatten(0, 1)
        mid = sorted(range(1, 98), key=lambda j: (-float(w[here[j], h]) if here[j] >= 0 else 1.0, j))
        keep = [0] + sorted(mid[:37]) + [98, 99]
        for xs in want.values():
            x, src = xs[0].flatten(0, 1), None
            src = x.clone()
            for j, s in enumerate(keep):
                if here[s] >= 0 and here[j] >= 0:
                    x[here[j], h] = src[here[s], h]
    assert handle(d).evict(bt.to(dev), ctx.to(dev), 40, sinks=1, recent=2).tolist() == [40]
    same(d, want)


def test_absent_pages_under_wide_tables(dev):
    """The same by transposed keys: absent pages within the sequences, of all their
    tokens, and behind them."""
    announce("evict: absent pages, tables of 9600 tokens")
    H, bs, width, budget, sinks, recent = 3, 16, 600, 70, 3, 9
    c, bt, ctx = make([9000, 300, 90], 2, H, 8, bs, scales=True, seed=14, width=width)
    g = torch.Generator().manual_seed(3)
    bt[0, torch.randperm(560, generator=g)[:40]] = -1
    bt[0, [0, 3, 561]] = 10 ** 6
    bt[1, 2], bt[1, 18], bt[2] = -1, 2 ** 31 - 1, -1
    d, want = on(dev, c), {n: [x.clone() for x in xs] for n, xs in c.items()}
    blocks = c["w"][0].shape[0]
    for b, n in enumerate(ctx.tolist()):
        t = torch.arange(n)
        page = bt[b, t // bs].long()
        here = torch.where((page >= 0) & (page < blocks), page * bs + t % bs, -1).tolist()
        for i in range(2):
            for h in range(H):
                w = c["w"][i].flatten(0, 1)[:, h].tolist()
                mid = sorted(range(sinks, n - recent), key=lambda j: (-w[here[j]] if here[j] >= 0 else 1.0, j))
                keep = list(range(sinks)) + sorted(mid[:budget - sinks - recent]) + list(range(n - recent, n))
                for name, xs in want.items():
                    x, src = xs[i].flatten(0, 1), c[name][i].flatten(0, 1)
                    for j, s in enumerate(keep):
                        if here[s] >= 0 and here[j] >= 0:
                            x[here[j], h] = src[here[s], h]
    new = handle(d).evict(bt.to(dev), ctx.to(dev), budget, sinks=sinks, recent=recent)
    assert new.tolist() == [70, 70, 70]
    same(d, want)


def test_turns_are_captured(dev):
    announce("evict: keys in turns, captured and replayed")
    c, bt, ctx = make([300, 900, 77], 3, 2, 8, 16, seed=15, width=(1 << 24) // 16)
    d, btd, ctxd = on(dev, c), bt.to(dev), ctx.to(dev)
    ev = handle(d)
    ev.evict(btd, ctxd, 60, sinks=2, recent=5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        out = ev.evict(btd, ctxd, 60, sinks=2, recent=5)
    g = torch.Generator().manual_seed(4)
    for turn in range(3):
        for n, xs in c.items():
            for x, y in zip(xs, d[n]):
                if x.dtype == torch.float32:
                    x.copy_(torch.rand(x.shape, generator=g))
                y.copy_(x)
        want = {n: [x.clone() for x in xs] for n, xs in c.items()}
        oracle(want, bt, ctx, 60, 2, 5)
        graph.replay()
        torch.cuda.synchronize()
        same(d, want)
        assert out.tolist() == [60, 60, 60]


def test_captured_replayed_and_on_another_stream(dev):
    announce("evict: captured twice, replayed on new weights, side stream")
    cases = []
    for seed, lens, width in ((11, [300, 200, 64], None), (12, [500, 90], 600)):
        c, bt, ctx = make(lens, 2, 2, 16, 16, seed=seed, width=width)
        d = on(dev, c)
        cases.append((c, bt, ctx, d, handle(d), bt.to(dev), ctx.to(dev)))
    outs, graphs = [], []
    for c, bt, ctx, d, ev, btd, ctxd in cases:
        ev.evict(btd, ctxd, 70, sinks=2, recent=9)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with graph_capture(graph):
            outs.append(ev.evict(btd, ctxd, 70, sinks=2, recent=9))
        graphs.append(graph)
    g = torch.Generator().manual_seed(2)
    side = torch.cuda.Stream()
    for turn in range(4):
        wants = []
        for c, bt, ctx, d, *_ in cases:
            for n, xs in c.items():
                for x, y in zip(xs, d[n]):
                    if x.dtype == torch.float32:
                        x.copy_(torch.rand(x.shape, generator=g))
                    y.copy_(x)
            want = {n: [x.clone() for x in xs] for n, xs in c.items()}
            oracle(want, bt, ctx, 70, 2, 9)
            wants.append(want)
        if turn < 3:
            for graph in graphs:
                graph.replay()
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for *_, ev, btd, ctxd in cases:
                    ev.evict(btd, ctxd, 70, sinks=2, recent=9)
            torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for (c, bt, ctx, d, *_), want, out in zip(cases, wants, outs):
            same(d, want)
            assert out.tolist() == ctx.clamp(max=70).tolist()


def test_trim_gives_pages_back(dev):
    """Rows let go of the pages past their tokens, shared pages stay with their
    other holders, and the pages can be handed out again."""
    announce("pages: trim")
    bs, pages = 16, 40
    pool = torch.zeros(pages, bs, 2, 8, device=dev)
    tables = torch.zeros(5, 10, dtype=torch.int32, device=dev)
    lens = torch.zeros(5, dtype=torch.int64, device=dev)
    p = mkv.PagePool(tables, lens, mkv.CachePages([pool]))

    def t(*x):
        return torch.tensor(x, dtype=torch.int64, device=dev)

    assert p.assign(t(0, 1, 2, -1, -1), t(100, 33, 160, 0, 0)).tolist() == [True] * 5
    lens.copy_(t(100, 33, 160, 0, 0))
    assert p.fork(2, [3]).tolist() == [True] * 5
    before, held = tables.clone(), p.held.tolist()
    assert held == [7, 3, 10, 10, 0]
    lens.copy_(t(40, 33, 96, 160, 5))
    p.trim()
    assert p.held.tolist() == [3, 3, 6, 10, 0]
    for r, h in enumerate(p.held.tolist()):
        assert tables[r, :h].tolist() == before[r, :h].tolist() and not any(tables[r, h:].tolist())
    refs = p.ref_counts.tolist()
    for page in before[0, 3:7].tolist():
        assert refs[page] == 0
    for i, page in enumerate(before[2, :10].tolist()):
        assert refs[page] == (2 if i < 6 else 1)
    assert sum(refs) == sum(p.held.tolist())
    lens.copy_(t(0, -3, 96, 160, 0))
    p.trim()
    assert p.held.tolist() == [0, 0, 6, 10, 0] and sum(p.ref_counts.tolist()) == 16
    lens.copy_(t(0, 0, 96, 160, 0))
    assert p.assign(t(0, 1, 2, 3, 4), t(160, 100, 96, 160, 5)).tolist() == [True] * 5
