"""GPU parity of the page table's step where its tables do not fit the
workgroup's LDS (more than 8192 entries), and where the free pages lie behind the
first sweep of the reference counts (16384 of them), against plain Python."""
from __future__ import annotations

import random

import pytest
import torch

import mkv
from conftest import announce
from mkv.decode_state import graph_capture
from test_gpu_pages import Table, caches

pytestmark = pytest.mark.gpu


def _pool(dev, rows, width, bs, N, taken=()):
    """An empty table, its plain counterpart, and pages with a holder besides."""
    ts = caches(dev, N, bs, [(torch.float32, (1,))], seed=rows)
    refs = torch.zeros(N, dtype=torch.int32)
    refs[list(taken)] = 1
    pool = mkv.PagePool(torch.zeros(rows, width, dtype=torch.int32, device=dev),
                        torch.zeros(rows, dtype=torch.int64, device=dev), mkv.CachePages(ts), ref_counts=refs.to(dev))
    t = Table(rows, width, bs, N, ts)
    t.refs = refs.tolist()
    return pool, t, ts


def _step(rng, t):
    parents, tokens = [], []
    for i in range(t.R):
        kind = rng.random()
        parents.append(i if kind < 0.45 else -1 if kind < 0.55 else rng.randrange(t.R))
        have = t.lens[parents[-1]] if parents[-1] >= 0 else 0
        tokens.append(rng.choice([0, have, have + 1, have + rng.randint(0, 4 * t.bs), rng.randint(0, t.W * t.bs),
                                  t.W * t.bs + 1]))
    return parents, tokens


def _written(rng, t):
    """The rows write into the pages they hold (not inside a page that others
    hold too)."""
    lens = [rng.randint(0, len(x) * t.bs) if rng.random() < 0.5 else n for x, n in zip(t.tables, t.lens)]
    t.lens = [n if n % t.bs == 0 or t.refs[x[n // t.bs]] == 1 else m for n, m, x in zip(lens, t.lens, t.tables)]
    return torch.tensor(t.lens)


@pytest.mark.parametrize("rows,width,bs,N", [(64, 256, 4, 9000), (1000, 20, 2, 7001), (1024, 9, 16, 3000), (8, 1500, 1, 5000),
                                             (33, 249, 2, 2500)])
def test_tables_past_the_lds(dev, rows, width, bs, N):
    announce(f"assign, {rows} rows of {width} pages of {bs}, {N} pages")
    assert rows * width > 8192
    rng = random.Random(width)
    pool, t, ts = _pool(dev, rows, width, bs, N)
    refused = copied = 0
    for step in range(7):
        parents, tokens = _step(rng, t)
        if step == 0:
            parents, tokens = [-1] * rows, [rng.randint(0, N * bs // rows) for _ in range(rows)]
        before = [list(x) for x in t.tables]
        want = t.assign(parents, tokens)
        refused += want.count(False)
        copied += sum(1 for i, p in enumerate(parents) if p >= 0 and want[i] and t.lens[i] % bs
                      and t.tables[i][t.lens[i] // bs] != before[p][t.lens[i] // bs])
        got = pool.assign(torch.tensor(parents, device=dev), torch.tensor(tokens, device=dev))
        assert got.tolist() == want
        t.check(pool, ts)
        pool.seq_lens.copy_(_written(rng, t))
    assert refused and (copied or bs == 1)
    pool.assign(torch.full((rows,), -1, device=dev))
    assert not pool.ref_counts.any() and not pool.held.any() and not pool.block_tables.any()


def test_large_tables_captured_and_replayed(dev):
    announce("assign, 64 rows of 256 pages, captured")
    rng = random.Random(4)
    pool, t, ts = _pool(dev, 64, 256, 4, 6000)
    parents, tokens = (torch.zeros(64, dtype=torch.int64, device=dev) for _ in range(2))
    pool.assign(torch.arange(64, device=dev))  # (nothing yet)
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        granted = pool.assign(parents, tokens)
    for step in range(5):
        p, n = _step(rng, t) if step else ([-1] * 64, [rng.randint(0, 300) for _ in range(64)])
        want = t.assign(p, n)
        parents.copy_(torch.tensor(p))
        tokens.copy_(torch.tensor(n))
        graph.replay()
        torch.cuda.synchronize()
        assert granted.tolist() == want, f"replay {step}"
        t.check(pool, ts)
        pool.seq_lens.copy_(_written(rng, t))


@pytest.mark.parametrize("N,free_from", [(20001, 16380), (33003, 32766), (16387, 16384), (50002, 49140), (32768, 32760)])
@pytest.mark.parametrize("rows,width", [(6, 12), (40, 300)])
def test_free_pages_behind_the_first_sweep(dev, N, free_from, rows, width):
    """All but a few of the lower pages have a holder besides; the pool runs out
    inside its last sweep."""
    announce(f"assign, {rows} rows of {width} pages, {N} pages, free from {free_from}")
    rng = random.Random(N + rows)
    spare = {rng.randrange(free_from) for _ in range(3)}
    pool, t, ts = _pool(dev, rows, width, 2, N, taken=[p for p in range(free_from) if p not in spare])
    free = N - free_from + len(spare)
    for step in range(4):
        if step == 0:  # some for every row
            parents, tokens = [-1] * rows, [2 * (free // rows) if i else 3 for i in range(rows)]
        elif step == 1:  # all there is, and more
            parents, tokens = list(range(rows)), [2 * width] * rows
        else:
            parents, tokens = _step(rng, t)
        want = t.assign(parents, tokens)
        got = pool.assign(torch.tensor(parents, device=dev), torch.tensor(tokens, device=dev))
        assert got.tolist() == want
        t.check(pool, ts)
        pool.seq_lens.copy_(_written(rng, t))


def test_a_refused_row_s_request_comes_first(dev):
    """Rows ask in their order: pages that a refused row asked for are not handed
    to the rows behind it, which need none or are refused as well."""
    announce("assign, a refused row ahead of rows that need pages")
    pool, t, ts = _pool(dev, 4, 8, 16, 4)
    parents, tokens = [0, 1, 2, 3], [16, 80, 16, 0]
    assert t.assign(parents, tokens) == [True, False, False, True]
    got = pool.assign(torch.tensor(parents, device=dev), torch.tensor(tokens, device=dev))
    assert got.tolist() == [True, False, False, True]
    t.check(pool, ts)
