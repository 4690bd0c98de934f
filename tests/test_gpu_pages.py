"""GPU parity of the page operations (copy, compact, assign) against plain
Python over lists and whole tensors: byte for byte, entry for entry."""
from __future__ import annotations

import random

import pytest
import torch

import mkv
from conftest import announce
from mkv.decode_state import DecodeMetadata, graph_capture

pytestmark = pytest.mark.gpu


def caches(dev, N, bs, tensors, seed=0):
    """One tensor a (dtype, trailing shape), random bytes."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for dtype, shape in tensors:
        size = torch.empty(0, dtype=dtype).element_size()
        flat = torch.randint(256, (N * bs * size * torch.Size(shape).numel(),), generator=g, dtype=torch.uint8)
        out.append(flat.view(dtype).view(N, bs, *shape).to(dev))
    return out


def same(a, b):
    return torch.equal(a.contiguous().view(-1).view(torch.uint8).cpu(), b.contiguous().view(-1).view(torch.uint8).cpu())


MIXES = {
    "bf16": [(torch.bfloat16, (8, 128))] * 4,
    "token": [(torch.int8, (2, 64)), (torch.float8_e4m3fn, (2, 64)), (torch.float32, (2,)), (torch.float32, (2,))],
    "odd": [(torch.float32, (3, 5)), (torch.bfloat16, (1, 2)), (torch.float32, (1,))],
    "layers": [(torch.bfloat16, (1, 64))] * 130,
}


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("bs", [1, 16, 256])
def test_copy(dev, mix, bs):
    announce(f"copy {mix} bs={bs}")
    N = 24
    ts = caches(dev, N, bs, MIXES[mix], seed=bs)
    want = [t.clone() for t in ts]
    rng = random.Random(bs)
    ids = rng.sample(range(N), 14)
    for w in want:
        w[ids[7:]] = w[ids[:7]]
    pages = mkv.CachePages(ts)
    pages.copy(ids[:7], ids[7:])
    assert all(same(a, b) for a, b in zip(ts, want))
    for dtype in (torch.int32, torch.int64):
        src, dst = (torch.tensor(x, dtype=dtype, device=dev) for x in (ids[:7], ids[7:]))
        for t in ts:
            t[ids[7:]] = 0
        pages.copy(src, dst)
        assert all(same(a, b) for a, b in zip(ts, want))
    # pages outside the pool, a page on itself, nothing at all
    pages.copy(torch.tensor([-1, N, 0, 3, 1 << 40], device=dev), torch.tensor([0, 1, -5, 3, 2], device=dev))
    pages.copy(torch.empty(0, dtype=torch.int64, device=dev), torch.empty(0, dtype=torch.int64, device=dev))
    pages.copy([], [])
    assert all(same(a, b) for a, b in zip(ts, want))


def test_copy_past_32_bits(dev):
    announce("copy large")
    t = torch.zeros(9000, 256, 8, 128, dtype=torch.int8, device=dev)
    assert t.numel() > 2 ** 31
    t[8999] = 7
    mkv.CachePages([t]).copy([8999], [8998])
    assert bool((t[8998] == 7).all()) and not bool(t[8997].any()) and not bool(t[0].any())


def compacted(ts, bt, prefix, accepted, bs):
    out = [t.clone() for t in ts]
    for b, row in enumerate(accepted):
        moves = []
        for j, a in enumerate(row):
            s, d = prefix[b] + a, prefix[b] + j
            if a < 0 or max(s, d) // bs >= len(bt[b]) or bt[b][s // bs] < 0 or bt[b][d // bs] < 0:
                continue
            moves.append((bt[b][s // bs], s % bs, bt[b][d // bs], d % bs))
        for o, t in zip(out, ts):
            for ps, rs, pd, rd in moves:
                o[pd, rd] = t[ps, rs]
    return out


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("cols", [1, 5, 40, 600])
def test_compact(dev, mix, cols):
    announce(f"compact {mix} {cols}")
    bs, B = 16, 5
    rng = random.Random(cols)
    prefix = [0, 15, 16, 37, 5]
    draft = cols + 9
    counts = [-(-(p + draft) // bs) for p in prefix]
    N = sum(counts) + 2
    ids = rng.sample(range(N), N)
    bt = []
    for n in counts:
        bt.append([ids.pop() for _ in range(n)] + [-1] * (max(counts) - n))
    accepted = [sorted(rng.sample(range(draft), rng.randint(0, cols))) for _ in range(B)]
    accepted[3] = rng.sample(range(draft), cols)  # any order: read before written
    accepted = [a + [-1] * (cols - len(a)) for a in accepted]
    if cols > 1:
        accepted[4] = [-1, 3] + [-1] * (cols - 2)  # a gap
        accepted[0][-1] = 1 << 30                  # outside the table
    ts = caches(dev, N, bs, MIXES[mix], seed=cols)
    want = compacted([t.cpu() for t in ts], bt, prefix, accepted, bs)
    pages = mkv.CachePages(ts)
    for dt in (torch.int64, torch.int32):
        new = caches(dev, N, bs, MIXES[mix], seed=cols)
        for t, n in zip(ts, new):
            t.copy_(n)
        acc = torch.tensor([[7] + a + [9] for a in accepted], dtype=dt, device=dev)[:, 1:-1]
        pages.compact(torch.tensor(bt, dtype=torch.int32, device=dev), torch.tensor(prefix, dtype=dt, device=dev), acc)
        assert all(same(a, b) for a, b in zip(ts, want))


def test_compact_leaves_bad_rows(dev):
    announce("compact bad")
    ts = caches(dev, 6, 16, MIXES["bf16"])
    want = [t.clone() for t in ts]
    pages = mkv.CachePages(ts)
    bt = torch.tensor([[0, 99], [1, -1], [2, 3]], dtype=torch.int32, device=dev)
    pages.compact(bt, torch.tensor([15, 15, -4], device=dev), torch.tensor([[1, 3]] * 3, device=dev))
    pages.compact(bt, torch.tensor([0, 0, 0], device=dev), torch.empty(3, 0, dtype=torch.int64, device=dev))
    pages.compact(bt, torch.tensor([1 << 50] * 3, device=dev), torch.tensor([[1, 3]] * 3, device=dev))
    assert all(same(a, b) for a, b in zip(ts, want))


class Table:
    """The page table's step in plain Python."""

    def __init__(self, rows, width, bs, N, ts):
        self.R, self.W, self.bs, self.N = rows, width, bs, N
        self.tables, self.lens, self.refs = [[] for _ in range(rows)], [0] * rows, [0] * N
        self.ts = [t.cpu() for t in ts]

    def assign(self, parents, tokens):
        R, bs = self.R, self.bs
        bad = [p >= R for p in parents]
        stays = [p == i or b for i, (p, b) in enumerate(zip(parents, bad))]
        new, lens = [], []
        for i, p in enumerate(parents):
            p = i if stays[i] else p
            lens.append(0 if p < 0 else self.lens[p])
            new.append([] if p < 0 else list(self.tables[p]) if stays[i] else self.tables[p][:-(-self.lens[p] // bs)])
        for i in range(R):
            if not stays[i]:
                for p in new[i]:
                    self.refs[p] += 1
        for i in range(R):
            if not stays[i]:
                for p in self.tables[i]:
                    self.refs[p] -= 1
        last = [new[i][lens[i] // bs] if lens[i] % bs else None for i in range(R)]
        refs = list(self.refs)
        free = [p for p in range(self.N) if refs[p] == 0]
        need, copies, grows = [], [], []
        for i in range(R):
            want = -(-tokens[i] // bs) if tokens[i] > 0 else 0
            alike = [r for r in range(R) if last[r] is not None and last[r] == last[i]]
            copy = last[i] is not None and refs[last[i]] > 1 and not (alike[0] == i and refs[last[i]] == len(alike))
            fits = not bad[i] and want <= self.W
            copies.append(copy)
            grows.append(max(want - len(new[i]), 0))
            need.append(copy + grows[i] if fits else None)
        granted, at = [], 0
        data = [t.clone() for t in self.ts]
        for i in range(R):
            n = need[i] or 0
            ok = need[i] is not None and (n == 0 or at + n <= len(free))
            granted.append(ok)
            mine, at = free[at:at + n], at + n
            if not ok:
                if not stays[i]:
                    for p in new[i]:
                        self.refs[p] -= 1
                    new[i], lens[i] = [], 0
                continue
            if copies[i]:
                fresh = mine.pop(0)
                for d, t in zip(data, self.ts):
                    d[fresh, :lens[i] % bs] = t[last[i], :lens[i] % bs]
                self.refs[last[i]] -= 1
                self.refs[fresh] += 1
                new[i][lens[i] // bs] = fresh
            for p in mine:
                self.refs[p] += 1
            new[i] += mine
        self.tables, self.lens, self.ts = new, lens, data
        return granted

    def check(self, pool, ts):
        assert pool.seq_lens.tolist() == self.lens
        assert pool.held.tolist() == [len(t) for t in self.tables]
        assert pool.block_tables.tolist() == [t + [0] * (self.W - len(t)) for t in self.tables]
        assert pool.ref_counts.tolist() == self.refs
        assert all(same(a, b) for a, b in zip(ts, self.ts))


@pytest.mark.parametrize("rows,width,bs,N", [(1, 1, 1, 1), (4, 3, 16, 9), (13, 9, 4, 40), (70, 20, 16, 500),
                                             (1000, 5, 2, 3000), (8, 700, 1, 20000)])
def test_assign_random_steps(dev, rows, width, bs, N):
    """Steps of forks, frees, growth and refusals from an empty table."""
    announce(f"assign {rows} {width} {bs} {N}")
    rng = random.Random(rows)
    ts = caches(dev, N, bs, [(torch.bfloat16, (1, 8)), (torch.float32, (1,))], seed=rows)
    pool = mkv.PagePool(torch.zeros(rows, width, dtype=torch.int32, device=dev),
                        torch.zeros(rows, dtype=torch.int64, device=dev), mkv.CachePages(ts))
    t = Table(rows, width, bs, N, ts)
    for step in range(8):
        parents, tokens = [], []
        for i in range(rows):
            kind = rng.random()
            parents.append(i if kind < 0.45 else -1 - rng.randrange(3) if kind < 0.6 else rng.randrange(rows))
            have = t.lens[parents[-1]] if parents[-1] >= 0 else 0
            tokens.append(rng.choice([0, -1, have, have + 1, have + rng.randint(0, 2 * bs + 3),
                                      rng.randint(0, width * bs), width * bs + 1]))
        if rows > 3 and step == 5:
            parents[2] = rows + 4  # no row: refused
        if step == 0:
            parents = [-1] * rows
        want = t.assign(parents, tokens)
        dt = torch.int32 if step % 2 else torch.int64
        got = pool.assign(torch.tensor(parents, dtype=dt, device=dev), torch.tensor(tokens, dtype=dt, device=dev))
        assert got.dtype == torch.bool and got.tolist() == want
        t.check(pool, ts)
        # the rows write into the pages they hold
        lens = [rng.randint(0, len(x) * bs) if rng.random() < 0.5 else n for x, n in zip(t.tables, t.lens)]
        # (a row's tokens never end inside a page that others hold too)
        lens = [n if n % bs == 0 or t.refs[x[n // bs]] == 1 else m for n, m, x in zip(lens, t.lens, t.tables)]
        t.lens = lens
        pool.seq_lens.copy_(torch.tensor(lens))
    assert pool.assign(torch.arange(rows, device=dev)).all()
    want = t.assign(list(range(rows)), [0] * rows)
    t.check(pool, ts)
    pool.assign(torch.full((rows,), -1, device=dev))
    assert not pool.ref_counts.any() and not pool.held.any() and not pool.block_tables.any()


def test_samples_of_one_prompt(dev):
    """fork and free by name over a DecodeMetadata: shared full pages, a copy
    of the last one for all but one row, a page kept by another holder."""
    announce("fork samples")
    bs, N = 16, 12
    meta = DecodeMetadata(4, 4, bs, N, dev)
    ts = caches(dev, N, bs, MIXES["token"])
    pool = mkv.PagePool(meta.block_tables, meta.seq_lens, mkv.CachePages(ts))
    pool.ref_counts[0] += 1  # not to be handed out
    assert pool.assign(torch.tensor([0, 1, -1, 3], device=dev), torch.tensor([0, 0, 40, 0], device=dev)).all()
    assert meta.block_tables[2].tolist() == [1, 2, 3, 0] and meta.seq_lens.tolist() == [0] * 4
    meta.seq_lens[2] = 35
    assert pool.fork(2, [0, 3]).all()
    assert meta.block_tables.tolist() == [[1, 2, 3, 0], [0] * 4, [1, 2, 4, 0], [1, 2, 5, 0]]
    assert pool.ref_counts.tolist() == [1, 3, 3, 1, 1, 1] + [0] * 6
    for t in ts:
        assert same(t[4, :3], t[3, :3]) and same(t[5, :3], t[3, :3])
    slot, ctx, _ = meta.step(4)
    assert ctx.tolist() == [36, 0, 36, 36] and slot.tolist() == [51, -1, 67, 83]
    pool.free([0, 2])
    assert pool.ref_counts.tolist() == [1, 1, 1, 0, 0, 1] + [0] * 6
    # the page table's own holder of a part-filled page: even its only row copies
    pool.ref_counts[5] += 1
    assert pool.assign(torch.arange(4, device=dev)).all()
    assert meta.block_tables[3].tolist() == [1, 2, 3, 0] and pool.ref_counts.tolist() == [1, 1, 1, 1, 0, 1] + [0] * 6


def test_assign_captured_and_replayed(dev):
    announce("assign graph")
    rows, width, bs, N = 6, 6, 4, 40
    ts = caches(dev, N, bs, [(torch.float32, (2, 4))], seed=3)
    pool = mkv.PagePool(torch.zeros(rows, width, dtype=torch.int32, device=dev),
                        torch.zeros(rows, dtype=torch.int64, device=dev), mkv.CachePages(ts))
    t = Table(rows, width, bs, N, ts)
    parents, tokens = torch.zeros(rows, dtype=torch.int64, device=dev), torch.zeros(rows, dtype=torch.int64, device=dev)
    steps = [([-1] * 6, [9, 5, 0, 17, 4, 0]), ([0, 0, 1, 3, 3, 3], [10, 11, 6, 18, 18, 20]),
             ([5, -1, 2, 2, 4, 0], [21, 0, 7, 7, 19, 24]), ([0, 1, 2, 3, 4, 5], [22, 3, 8, 8, 20, 24])]
    pool.assign(torch.arange(rows, device=dev))  # (nothing yet)
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        granted = pool.assign(parents, tokens)
    for p, n in steps:
        want = t.assign(p, n)
        parents.copy_(torch.tensor(p))
        tokens.copy_(torch.tensor(n))
        graph.replay()
        torch.cuda.synchronize()
        assert granted.tolist() == want
        t.check(pool, ts)
        t.lens = [max(x - 1, 0) for x in n]
        pool.seq_lens.copy_(torch.tensor(t.lens))
