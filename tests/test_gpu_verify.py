"""GPU tests of the verification of drafted tokens (mkv_verify_drafts).

Oracle: the walk in float64 on the CPU, node by node, from the definition.  What a
walk decides is compared where it is decided by more than the kernel's rounding
(1e-3 of the compared values; nearly all sequences), whole numbers exactly.
"""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce
from mkv.decode_state import graph_capture

pytestmark = pytest.mark.gpu

# Acceptance: p's and q's exponents are products (x - m) log2(e) / T of |t| <= 64 here
# with four roundings of 2^-24, so each e^ is off by 64 * 4 * 2^-24 ln 2 = 1.06e-5,
# the sums by no more; p / q has four of them.
RTOL = 5e-5
CLEAR = 1e-3


def make(dtype, sizes, vocab, kids, drawn, temps, seed=0, masked=0.0, spread=3.0, extra=0):
    g = torch.Generator().manual_seed(seed)
    total, B = sum(sizes) + extra, len(sizes)
    x = torch.randn(total, vocab, generator=g) * spread
    d = (x + torch.randn(total, vocab, generator=g)).to(dtype)
    x = x.to(dtype)
    if masked:
        x[:, torch.rand(vocab, generator=g) < masked] = -math.inf
        x[:, vocab // 2] = 0.25
    parents, ids = torch.zeros(total, dtype=torch.int64), torch.randint(0, vocab, (total,), generator=g)
    r = 0
    for n, t in zip(sizes, temps):
        for i in range(n):
            if i:
                p = i - 1 if kids == 1 else int(torch.randint(max(0, i - kids), i, (1,), generator=g))
                parents[r + i] = p
                row = d[r + p].double() / (t or 1e-6)
                if drawn:
                    ids[r + i] = int(torch.multinomial(torch.softmax(row, -1), 1, generator=g))
                else:
                    before = int((parents[r + 1:r + i] == p).sum())
                    ids[r + i] = int(torch.sort(row, descending=True, stable=True).indices[before % vocab])
            else:
                parents[r] = -1
        r += n
    cu = torch.tensor([0] + list(sizes), dtype=torch.int32).cumsum(0).to(torch.int32)
    return dict(logits=x, token_ids=ids, cu_seqlens_q=cu, uniforms=torch.rand(total, generator=g),
                noise=torch.empty(B, vocab).exponential_(generator=g), max_nodes=max(list(sizes) + [1]),
                parents=None if kids == 1 else parents, draft_logits=d if drawn else None,
                temperatures=torch.tensor(temps, dtype=torch.float32))


def _dist(row, t):
    """(probabilities, whether greedy)"""
    row = row.double()
    order = torch.where(torch.isnan(row), math.inf, row)
    if t <= 1e-30 or not bool(torch.isfinite(row.max())) or bool(torch.isnan(row).any()):
        top = torch.where(torch.isnan(row), 2.0, torch.where(order == order.max(), 1.0, 0.0))
        p = torch.zeros_like(row)
        p[int((top == top.max()).nonzero()[0])] = 1
        return p, True
    return torch.softmax(row / t, -1), False


def oracle(c):
    """paths, next tokens, acceptance, and which sequences are decided clearly"""
    paths, nexts, sure = [], [], []
    acceptance = torch.full((c["logits"].shape[0],), math.nan, dtype=torch.float64)
    V = c["logits"].shape[1]
    cu = c["cu_seqlens_q"].tolist()
    for s in range(len(cu) - 1):
        r, n = cu[s], min(cu[s + 1] - cu[s], c["max_nodes"])
        acceptance[cu[s]:cu[s + 1]] = 0
        t = 1.0 if c["temperatures"] is None else float(c["temperatures"][s])
        if n == 0:
            paths.append([])
            nexts.append(-1)
            sure.append(True)
            continue
        acceptance[r] = 1
        parents = list(range(-1, n - 1)) if c["parents"] is None else c["parents"][r:r + n].tolist()
        clear, cur, path = True, 0, [0]
        dists = {}

        def dist(i):
            if i not in dists:
                p, greedy = _dist(c["logits"][r + i], t)
                q = None
                if c["draft_logits"] is not None and not greedy:
                    q, bad = _dist(c["draft_logits"][r + i], t)
                    q = None if bad else q
                dists[i] = p, q, greedy
            return dists[i]

        for i in range(1, n):
            x, a = int(c["token_ids"][r + i]), parents[i]
            if 0 <= a < i and 0 <= x < V:
                p, q, _ = dist(a)
                acceptance[r + i] = min(1.0, float(p[x] if q is None else p[x] / q[x]))
        rest = dist(0)[0].clone()
        for i in range(1, n):
            if parents[i] != cur:
                continue
            p, q, greedy = dist(cur)
            x = int(c["token_ids"][r + i])
            inside = 0 <= x < V
            left, u = (float(rest[x]) if inside else 0.0), float(c["uniforms"][r + i])
            bar = u * (1.0 if q is None else float(q[x]) if inside else 0.0)
            take = left > 0 if greedy else inside and bar < left
            if not greedy and inside:
                clear &= abs(bar - left) > CLEAR * max(bar, left) or (left == 0 and q is None)
            if take:
                cur = i
                path.append(i)
                rest = dist(i)[0].clone()
            elif not greedy:
                if q is None:
                    if inside:
                        rest[x] = 0
                else:
                    near = (rest - q).abs() <= 1e-6 * q  # (what the rounding leaves)
                    rest = torch.where(near, 0, (rest - q).clamp(min=0))
                total = float(rest.sum())
                clear &= total > 1e-3
                rest = rest / total if total > 0 else rest
        p, q, greedy = dist(cur)
        if greedy:
            nexts.append(int(p.argmax()))
        else:
            value = rest / c["noise"][s].double()
            top = torch.sort(value, descending=True, stable=True)
            nexts.append(int(top.indices[0]))
            if V > 1:
                clear &= bool(top.values[1] < top.values[0] * (1 - CLEAR))
        paths.append(path)
        sure.append(bool(clear))
    return paths, nexts, acceptance, sure


def on(dev, c):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def check(r, c, least=0.9):
    paths, nexts, acceptance, sure = oracle(c)
    got, count, token = r.accepted.cpu().tolist(), r.num_accepted.cpu().tolist(), r.next_tokens.cpu().tolist()
    assert r.accepted.shape == (len(paths), c["max_nodes"])
    for s, (path, nxt, clear) in enumerate(zip(paths, nexts, sure)):
        if clear:
            want = path + [-1] * (c["max_nodes"] - len(path))
            assert (got[s], count[s], token[s]) == (want, len(path), nxt), f"sequence {s}"
    assert sum(sure) >= least * len(sure), f"{sum(sure)} of {len(sure)} sequences are decided clearly"
    have = r.acceptance.cpu().double()
    rows = ~torch.isnan(acceptance)
    assert bool(((have - acceptance).abs() <= RTOL * acceptance + 1e-12)[rows].all())
    return paths


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [2, 33, 513, 8191, 8193, 20011])
@pytest.mark.parametrize("kids,drawn", [(1, True), (1, False), (3, True), (4, False)])
def test_walks(dev, dtype, vocab, kids, drawn):
    announce(f"verify: {dtype}, {vocab} tokens, up to {kids} children or so, drawn {drawn}")
    sizes = [1, 2, 5, 9, 17, 3, 30, 4, 12, 8, 7, 6] if vocab < 9000 else [1, 5, 14, 2]
    temps = [1.0, 0.0, 0.7, 1.3, 1.0, 0.6, 1.0, 0.0, 2.0, 1.0, 0.9, 1.0][:len(sizes)]
    # (two tokens leave little after a rejection: most such sequences still decide clearly)
    c = make(dtype, sizes, vocab, kids, drawn, temps, seed=vocab + kids)
    paths = check(mkv.verify_drafts(**on(dev, c)), c, least=0.7)
    # (four sequences of a large vocabulary: the oracle's own walks may all end at once)
    assert vocab > 9000 or any(len(p) > 1 for p in paths)


def test_a_full_vocabulary_and_many_sequences(dev):
    announce("verify: 151936 tokens; 150 sequences")
    c = make(torch.bfloat16, [9, 5], 151936, 1, True, [1.0, 0.8], seed=1)
    check(mkv.verify_drafts(**on(dev, c)), c, least=0.5)
    sizes = [1 + i % 6 for i in range(150)]
    c = make(torch.float32, sizes, 300, 2, True, [[1.0, 0.0, 0.5][i % 3] for i in range(150)], seed=2)
    check(mkv.verify_drafts(**on(dev, c)), c)


def test_siblings_over_a_full_vocabulary(dev):
    """Trees drawn from the draft over 151,936 tokens, their uniforms high: siblings
    behind one, two and three rejections, each with the sum of what is left."""
    announce("verify: drawn trees of four children over 151936 tokens")
    sizes = [5, 13, 5, 9, 5, 21]
    c = make(torch.bfloat16, sizes, 151936, 4, True, [1.0, 0.8, 1.2, 1.0, 0.7, 1.0], seed=6)
    for s, n in enumerate(sizes):
        r = int(c["cu_seqlens_q"][s])
        g = torch.Generator().manual_seed(s)
        for i in range(1, n):
            p = (i - 1) // 4
            c["parents"][r + i] = p
            row = torch.softmax(c["draft_logits"][r + p].double() / float(c["temperatures"][s]), -1)
            c["token_ids"][r + i] = int(torch.multinomial(row, 1, generator=g))
    c["uniforms"] = 0.7 + 0.3 * c["uniforms"]
    check(mkv.verify_drafts(**on(dev, c)), c, least=0.5)


@pytest.mark.parametrize("drawn", [True, False])
def test_masked_tokens_ties_and_odd_rows(dev, drawn):
    """A grammar's -inf, rows with NaN, +inf or nothing, equal logits, equal
    siblings, tokens outside the vocabulary, parents that are none, sequences
    without nodes and rows behind the last one."""
    announce(f"verify: odd rows, drawn {drawn}")
    sizes = [6, 0, 6, 6, 6, 0, 6, 6]
    c = make(torch.bfloat16, sizes, 1000, 2, drawn, [1.0] * 6 + [0.0, 1.0], seed=3, masked=0.6, extra=3)
    c["logits"][1, 17] = math.nan
    c["logits"][6, 18] = math.inf
    c["logits"][6, 900] = math.inf
    c["logits"][12] = -math.inf
    c["logits"][18] = 0.5                       # all alike
    c["logits"][26, 30] = c["logits"][26, 40] = 60.0  # greedy's ties
    if drawn:
        c["draft_logits"][2, 5] = math.nan
        c["draft_logits"][13] = -math.inf
    c["token_ids"][3], c["token_ids"][9], c["token_ids"][33] = -5, 1000, 2 ** 40
    c["token_ids"][19:24] = 77                  # (one token five times)
    c["parents"][20], c["parents"][22], c["parents"][34] = 5, -1, 2 ** 35
    c["parents"][30:32] = 0
    got = mkv.verify_drafts(**on(dev, c))
    check(got, c, least=0.6)
    chain = dict(c, parents=None)
    check(mkv.verify_drafts(**on(dev, chain)), chain, least=0.6)
    short = dict(c, max_nodes=3)
    check(mkv.verify_drafts(**on(dev, short)), short, least=0.6)
    for rows in (0, 1):
        none = dict(c, logits=c["logits"][:rows], token_ids=c["token_ids"][:rows], uniforms=c["uniforms"][:rows],
                    parents=c["parents"][:rows], draft_logits=c["draft_logits"][:rows] if drawn else None,
                    cu_seqlens_q=torch.tensor([0, 0, rows], dtype=torch.int32), noise=c["noise"][:2],
                    temperatures=None)
        check(mkv.verify_drafts(**on(dev, none)), none, least=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_index_types(dev, dtype):
    announce(f"verify: strided, unaligned and 32-bit inputs, {dtype}")
    c = make(dtype, [5, 8, 3], 777, 3, True, [1.0, 0.9, 0.0], seed=5)
    d = on(dev, c)
    want = mkv.verify_drafts(**d)
    check(want, c, least=0.6)

    def inside(t, left, right):
        big = torch.full((t.shape[0], t.shape[1] + left + right), 50.0, dtype=t.dtype, device=dev)
        big[:, left:left + t.shape[1]] = t
        return big[:, left:left + t.shape[1]]

    for left, right in ((1, 2), (3, 0), (5, 8)):
        e = dict(d, logits=inside(d["logits"], left, right), draft_logits=inside(d["draft_logits"], right, left),
                 noise=inside(d["noise"], left, left), token_ids=d["token_ids"].int(), parents=d["parents"].int())
        got = mkv.verify_drafts(**e)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = dict(d, logits=d["logits"].t().contiguous().t(), cu_seqlens_q=d["cu_seqlens_q"].long())
    assert all(torch.equal(a, b) for a, b in zip(mkv.verify_drafts(**turned), want))


@pytest.mark.parametrize("kids,drawn", [(1, True), (1, False), (3, True), (3, False)])
def test_tokens_follow_the_target_s_distribution(dev, kids, drawn):
    """40,000 sequences with the same two rows: the first new token of each (a
    child accepted, or the token drawn) is distributed as the target's, whatever
    the draft's.  Frequencies are within five standard deviations."""
    announce(f"verify: the distribution of what is generated, {kids} children, drawn {drawn}")
    g = torch.Generator().manual_seed(8)
    N, V, n = 40000, 11, 1 + kids
    p, q = torch.softmax(torch.randn(V, generator=g) * 1.5, -1), torch.softmax(torch.randn(V, generator=g), -1)
    logits = p.log().repeat(N * n, 1)
    if drawn:
        kid = torch.multinomial(q, N * kids, replacement=True, generator=g).reshape(N, kids)
    else:
        kid = q.argsort(descending=True)[:kids].expand(N, kids)
    ids = torch.cat([torch.zeros(N, 1, dtype=torch.int64), kid], 1).flatten()
    c = dict(logits=logits, token_ids=ids, cu_seqlens_q=torch.arange(0, N * n + 1, n, dtype=torch.int32),
             uniforms=torch.rand(N * n, generator=g), noise=torch.empty(N, V).exponential_(generator=g), max_nodes=n,
             parents=torch.tensor([-1] + [0] * kids).repeat(N), draft_logits=q.log().repeat(N * n, 1) if drawn else None)
    r = mkv.verify_drafts(**on(dev, c))
    first = torch.where(r.num_accepted > 1, ids.to(dev).reshape(N, n).gather(1, r.accepted[:, 1:2].clamp(min=0))[:, 0],
                        r.next_tokens)
    freq = torch.bincount(first.cpu(), minlength=V).double() / N
    sd = (p.double() * (1 - p.double()) / N).sqrt()
    assert bool(((freq - p.double()).abs() <= 5 * sd).all()), (freq, p)


def test_captured_and_on_a_side_stream(dev):
    """Two captured graphs, replayed with eager calls in between and new inputs
    in place: each replay as the eager call."""
    announce("verify: captured twice, replayed, side stream")
    cases = [on(dev, make(torch.bfloat16, [5, 9, 3], 9000, 1, True, [1.0, 0.0, 0.8], seed=11)),
             on(dev, make(torch.float32, [4, 7], 600, 3, False, [1.0, 0.5], seed=12))]
    outs, graphs = [], []
    for c in cases:
        mkv.verify_drafts(**c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with graph_capture(graph):
            outs.append(mkv.verify_drafts(**c))
        graphs.append(graph)
    gen = torch.Generator(device=dev).manual_seed(4)
    for turn in range(4):
        for c in cases:
            c["uniforms"].uniform_(generator=gen)
            c["noise"].exponential_(generator=gen)
        for graph in graphs:
            graph.replay()
        want = [mkv.verify_drafts(**c) for c in cases]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), f"replay {turn}"
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mkv.verify_drafts(**cases[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, mkv.verify_drafts(**cases[0])))
