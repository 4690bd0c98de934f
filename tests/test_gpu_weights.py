"""GPU tests of the attention weights accumulated beside the cache
(mkv_paged_weights) against the definition in float64 on the CPU.

Tolerance: the products of a score are exact, the sum of its D terms is fp32: off by
at most D 2^-24 times the sum of their sizes, here below 128 * 2^-24 * 18 = 1.4e-4
(1.5 x unit queries and unit keys give 11 on average at D = 128, scaled).  The score's
other roundings are below 2^-20.  A weight has that from its score and from its
normaliser, 2.8e-4 in all; sums of weights add 2^-22, decay another rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce
from mkv import workloads as W
from mkv.decode_state import graph_capture

pytestmark = pytest.mark.gpu

RTOL = 3e-4
CACHES = {"fp32": (torch.float32, torch.float32, "auto"), "bf16": (torch.bfloat16, torch.bfloat16, "auto"),
          "fp16": (torch.float16, torch.float16, "auto"), "fp8": (torch.float8_e4m3fn, torch.bfloat16, "fp8_per_tensor"),
          "fp8_q16": (torch.float8_e4m3fn, torch.float16, "fp8_per_tensor"),
          "fp8_token": (torch.float8_e4m3fn, torch.bfloat16, "fp8_per_token_head"),
          "fp8_token_q16": (torch.float8_e4m3fn, torch.float16, "fp8_per_token_head"),
          "int8_token": (torch.int8, torch.bfloat16, "int8_per_token_head"),
          "int8_token_q16": (torch.int8, torch.float16, "int8_per_token_head")}


def make(fmt, rows, ctx, Hq, Hkv, D, bs, seed=0, spare=3):
    """rows: of each sequence, or None for one each without cu_seqlens_q."""
    g = torch.Generator().manual_seed(seed)
    cdt, qdt, mode = CACHES[fmt]
    lens = torch.tensor(ctx, dtype=torch.int64)
    blocks = sum(-(-n // bs) for n in ctx) + spare
    bt = W.fragmented_block_tables(lens, bs, blocks, g)
    k = torch.randn(blocks, bs, Hkv, D, generator=g)
    scale = None
    if mode == "fp8_per_tensor":
        scale = torch.tensor([0.013])
        k = (k / scale).clamp(-448, 448)
    elif mode != "auto":
        top = 127.0 if cdt == torch.int8 else 448.0
        scale = (torch.rand(blocks, bs, Hkv, generator=g) * 0.5 + 0.75) * 3 / top
        k = (k * top / 3).clamp(-top, top)
        k = k.round() if cdt == torch.int8 else k
    total = len(ctx) if rows is None else sum(rows)
    return dict(query=(torch.randn(total, Hq, D, generator=g) * 1.5).to(qdt), k_cache=k.to(cdt),
                weights=torch.rand(blocks, bs, Hkv, generator=g), block_tables=bt, context_lens=lens,
                scale=1 / math.sqrt(D), num_heads=Hq, num_kv_heads=Hkv, head_dim=D, block_size=bs,
                cu_seqlens_q=None if rows is None else torch.tensor([0] + list(rows)).cumsum(0).to(torch.int32),
                k_scale=scale, kv_cache_dtype=mode)


def on(dev, c):
    return {n: v.to(dev) if isinstance(v, torch.Tensor) else v for n, v in c.items()}


def oracle(c, decay):
    """(weights, what the call adds), float64"""
    w, add = c["weights"].double().flatten(0, 1).clone(), torch.zeros_like(c["weights"].double()).flatten(0, 1)
    Hkv, bs, D = c["num_kv_heads"], c["block_size"], c["head_dim"]
    G, k = c["num_heads"] // Hkv, c["k_cache"].double()
    if c["k_scale"] is not None:
        k = k * (c["k_scale"].double() if c["k_scale"].numel() == 1 else c["k_scale"].double()[..., None])
    k = k.flatten(0, 1)
    B = len(c["context_lens"])
    cu = list(range(B + 1)) if c["cu_seqlens_q"] is None else c["cu_seqlens_q"].tolist()
    blocks = c["k_cache"].shape[0]
    for b in range(B):
        n, length = cu[b + 1] - cu[b], int(c["context_lens"][b])
        t = torch.arange(min(length, c["block_tables"].shape[1] * bs))
        page = c["block_tables"][b, t // bs].long()
        here = (page >= 0) & (page < blocks)
        t, slots = t[here], (page * bs + t % bs)[here]
        old = (t < length - n)[:, None]
        w[slots] = torch.where(old & (decay != 0), decay * w[slots], 0.0)
        if n == 0 or t.numel() == 0:
            continue
        q = c["query"][cu[b]:cu[b + 1]].double()
        hidden = t[None] > (length - n + torch.arange(n))[:, None]
        for h in range(c["num_heads"]):
            s = q[:, h] @ k[slots][:, h // G].t() * c["scale"]
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            p = torch.where(hidden, 0.0, p)  # (a row that sees nothing: NaN there)
            add[slots, h // G] += p.sum(0)
    return (w + add).reshape(c["weights"].shape), add.reshape(c["weights"].shape)


def check(dev, c, decay=1.0):
    d = on(dev, c)
    got = mkv.paged_attention_weights(**d, decay=decay)
    assert got.data_ptr() == d["weights"].data_ptr()
    want, add = oracle(c, decay)
    have = got.cpu().double()
    tol = RTOL * add + 2.0 ** -22 * want.abs() + 1e-30
    bad = ~((have - want).abs() <= tol) & ~(torch.isnan(have) & torch.isnan(want))
    assert not bool(bad.any()), (f"{int(bad.sum())} entries off, at most {float(((have - want).abs() / tol)[bad].max()):.1f} "
                                 f"times the tolerance; first {bad.nonzero()[0].tolist()}")
    return got


SHAPES = [(8, 8, 128, 16), (16, 8, 128, 256), (6, 2, 64, 32), (32, 8, 128, 32), (8, 1, 64, 16), (16, 1, 128, 16), (9, 3, 64, 64)]


@pytest.mark.parametrize("fmt", list(CACHES))
@pytest.mark.parametrize("Hq,Hkv,D,bs", SHAPES)
def test_decode(dev, fmt, Hq, Hkv, D, bs):
    announce(f"weights: decode, {fmt}, {Hq}/{Hkv} heads of {D}, blocks of {bs}")
    for decay in (1.0, 0.0):
        check(dev, make(fmt, None, [1, 0, 15, 16, 17, 250, 700, 64, 129], Hq, Hkv, D, bs, seed=Hq + D), decay)


@pytest.mark.parametrize("fmt", list(CACHES))
@pytest.mark.parametrize("Hq,Hkv,D,bs", SHAPES)
def test_chunks(dev, fmt, Hq, Hkv, D, bs):
    announce(f"weights: chunks, {fmt}, {Hq}/{Hkv} heads of {D}, blocks of {bs}")
    for rows, ctx, decay in (([1, 5, 0, 33, 70, 3, 1], [1, 300, 40, 33, 131, 2, 520], 0.9),
                             ([150, 90], [150, 700], 1.0), ([17], [260], 0.0)):
        check(dev, make(fmt, rows, ctx, Hq, Hkv, D, bs, seed=Hq + len(rows)), decay)


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8", "int8_token"])
def test_long_contexts(dev, fmt):
    announce(f"weights: split contexts, {fmt}")
    for Hq, Hkv, D in ((8, 2, 128), (24, 3, 64)):
        check(dev, make(fmt, None, [9000, 5, 4097, 1024], Hq, Hkv, D, 16, seed=3), 0.5)
        check(dev, make(fmt, [3, 20, 1], [9000, 2100, 4097], Hq, Hkv, D, 32, seed=4), 0.5)


def test_many_sequences(dev):
    announce("weights: 150 sequences")
    ctx = [1 + 7 * i % 97 for i in range(150)]
    check(dev, make("bf16", None, ctx, 4, 2, 128, 16, seed=5))
    rows = [i % 4 for i in range(150)]
    check(dev, make("bf16", rows, [n + r for n, r in zip(ctx, rows)], 4, 2, 128, 16, seed=6))


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "int8_token"])
def test_runs_of_units_cross_sequences(dev, fmt):
    """More units of keys than workgroups: each takes several, of several sequences,
    some of them empty."""
    announce(f"weights: 140 sequences of 16 KV heads, {fmt}")
    ctx = [0 if i % 5 == 3 else 1 + 61 * i % 700 for i in range(140)]
    rows = [min(n, 1 + i % 7) if i % 4 else 0 for i, n in enumerate(ctx)]
    check(dev, make(fmt, rows, ctx, 32, 16, 64, 16, seed=17), 0.5)


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8_token"])
def test_short_sequences(dev, fmt):
    """A few tokens each: pieces of the rows' work that hold none of a block's keys."""
    announce(f"weights: 64 sequences of 3 to 80 tokens, {fmt}")
    for Hq, Hkv in ((6, 2), (16, 16)):
        rows = [3 + i % 2 for i in range(64)]
        check(dev, make(fmt, rows, [n + i * 7 % 78 for i, n in enumerate(rows)], Hq, Hkv, 64, 16, seed=18), 0.5)


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8"])
@pytest.mark.parametrize("width", [1008, 1024, 1040, 4080, 4096, 4112])
def test_widths_at_which_a_context_is_split(dev, fmt, width):
    announce(f"weights: a table of {width} tokens, {fmt}")
    for Hq in (4, 10):  # (a group of up to four, and more)
        check(dev, make(fmt, None, [width, width - 15, 3], Hq, 2, 128, 16, seed=width), 0.5)


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8_token"])
def test_a_prompt_s_rows(dev, fmt):
    """Hundreds of rows of each sequence: every form of the row blocks."""
    announce(f"weights: whole prompts and chunks of them, {fmt}")
    check(dev, make(fmt, [600], [600], 4, 2, 128, 16, seed=7))
    check(dev, make(fmt, [300, 513, 70], [1500, 513, 71], 8, 2, 64, 32, seed=8), 0.9)
    check(dev, make(fmt, [100, 64], [900, 64], 2, 2, 128, 256, seed=9))


@pytest.mark.parametrize("rows", [None, [1, 4, 30]])
def test_tables_with_holes_and_wide_ones(dev, rows):
    """Absent pages are neither seen nor written; tables far wider than the
    contexts (so wide that kept scores would not fit) give the same; contexts
    longer than the table; rows more than the context has tokens."""
    announce(f"weights: absent pages, wide and narrow tables, rows {rows}")
    c = make("bf16", rows, [300, 77, 900], 8, 2, 128, 16, seed=10)
    c["block_tables"][0, 3], c["block_tables"][2, 40], c["block_tables"][2, 0] = -1, 10 ** 6, -1
    check(dev, c)
    pad = 4300000 // 16
    wide = dict(c, block_tables=torch.cat([c["block_tables"], torch.full((3, pad), -1, dtype=torch.int32)], 1))
    wide = dict(wide, num_kv_heads=2)
    check(dev, wide)
    many = make("bf16", rows, [300, 77, 900], 16, 8, 64, 16, seed=11)
    check(dev, dict(many, block_tables=torch.cat([many["block_tables"], torch.zeros(3, pad, dtype=torch.int32)], 1)))
    check(dev, dict(c, block_tables=c["block_tables"][:, :10].contiguous()))
    check(dev, dict(c, context_lens=torch.tensor([3, 2, 20])))
    if rows:
        check(dev, dict(c, cu_seqlens_q=torch.tensor([0, 10, 10, 35], dtype=torch.int32),
                        context_lens=torch.tensor([4, 0, 25])))


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "fp8_token"])
@pytest.mark.parametrize("Hq,Hkv,tokens", [(8, 4, 1 << 20), (10, 2, 1 << 20), (10, 2, 4300000), (2, 1, 17000000)])
def test_scores_that_are_kept_in_turns(dev, fmt, Hq, Hkv, tokens):
    """Tables so wide that the scores of some (sequence, KV head) pairs are kept at a
    time, and ones under which a single pair's are not kept at all."""
    announce(f"weights: decode, {fmt}, {Hq}/{Hkv} heads, tables of {tokens} tokens")
    c = make(fmt, None, [2900, 1, 0, 1025, 64], Hq, Hkv, 64, 16, seed=19)
    pad = torch.full((5, tokens // 16 - c["block_tables"].shape[1]), -1, dtype=torch.int32)
    check(dev, dict(c, block_tables=torch.cat([c["block_tables"], pad], 1)), 0.5)


def test_turns_are_captured(dev):
    announce("weights: scores kept in turns, captured and replayed")
    c = make("fp8", None, [2900, 1, 0, 1025, 64], 10, 2, 64, 16, seed=20)
    pad = torch.full((5, (1 << 20) // 16 - c["block_tables"].shape[1]), -1, dtype=torch.int32)
    d = on(dev, dict(c, block_tables=torch.cat([c["block_tables"], pad], 1)))
    mkv.paged_attention_weights(**d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with graph_capture(graph):
        mkv.paged_attention_weights(**d)
    for turn in range(3):
        before = d["weights"].clone()
        graph.replay()
        want = mkv.paged_attention_weights(**dict(d, weights=before))
        torch.cuda.synchronize()
        assert torch.equal(d["weights"], want), f"replay {turn}"


def test_sequences_that_share_pages_take_turns(dev):
    """Forks over shared pages, a call each: what every one of them gives is there."""
    announce("weights: two sequences over the same pages, a call each")
    c = make("bf16", None, [70, 70], 8, 2, 128, 16, seed=21)
    c["block_tables"][1, :4] = c["block_tables"][0, :4]
    d, w = on(dev, c), c["weights"]
    for b in range(2):
        one = dict(query=c["query"][b:b + 1], block_tables=c["block_tables"][b:b + 1], context_lens=c["context_lens"][b:b + 1])
        mkv.paged_attention_weights(**dict(d, **on(dev, one)), decay=0.5)
        w, add = oracle(dict(c, weights=w, **one), 0.5)
    assert float((d["weights"].cpu().double() - w).abs().max()) <= RTOL * 4 * 2 + 2.0 ** -21


@pytest.mark.parametrize("rows", [None, [300, 0, 33, 520, 7, 1]])
@pytest.mark.parametrize("fmt", ["fp32", "bf16"])
def test_lengths_far_past_the_table(dev, fmt, rows):
    """A length that no table holds: its rows see what the table has."""
    announce(f"weights: lengths up to 2^62, {fmt}, rows {rows}")
    c = make(fmt, rows, [700, 90, 33, 520, 64, 9], 16, 2, 64, 16, seed=22)
    c["context_lens"] = torch.tensor([2 ** 62, 2 ** 45 + 12345, 33, 2 ** 50 - 1, 2 ** 44, 9])
    check(dev, c, 0.5)


def test_values_that_are_not_finite(dev):
    """A NaN key reaches what the rows that see it see, and nothing else; tokens
    that no row sees change nothing; the entries of new tokens may hold anything."""
    announce("weights: NaN and infinities")
    for rows in (None, [40]):
        c = make("bf16", rows, [200], 4, 2, 128, 16, seed=12)
        slots = [int(c["block_tables"][0, t // 16]) * 16 + t % 16 for t in range(208)]
        new = 1 if rows is None else 40
        w = c["weights"].flatten(0, 1)
        w[slots[200 - new:200]] = math.nan
        c["k_cache"].flatten(0, 1)[slots[200:208]] = math.nan  # (behind the context)
        got = check(dev, c)
        assert not bool(torch.isnan(got.cpu().flatten(0, 1)[slots[:200]]).any())
        c["k_cache"].flatten(0, 1)[slots[190], 1, 5] = math.nan
        # row i of 40 sees token 190 from i = 30 on: those rows are NaN in all they see,
        # so head 1's sums are NaN up to the last row's token; head 0's are not
        got = mkv.paged_attention_weights(**on(dev, c)).cpu().flatten(0, 1)
        assert bool(torch.isnan(got[slots[:200], 1]).all()) and not bool(torch.isnan(got[slots[:200], 0]).any())
        if rows:
            # only the rows ahead of it: as without it
            early = dict(c, query=c["query"][:30], cu_seqlens_q=torch.tensor([0, 30], dtype=torch.int32),
                         context_lens=torch.tensor([190]))
            check(dev, early)


def test_strides_index_types_and_streams(dev):
    announce("weights: strided queries and tables, int32 lengths, another stream, captured twice")
    cases = [make("bf16", None, [300, 700, 64], 8, 2, 128, 16, seed=13), make("fp8", [20, 7], [90, 400], 8, 4, 64, 32, seed=14),
             make("fp32", None, [5000, 33], 4, 4, 128, 16, seed=15)]
    for c in cases:
        d = on(dev, c)
        want = mkv.paged_attention_weights(**dict(d, weights=d["weights"].clone()))
        big = torch.zeros(d["query"].shape[0], d["query"].shape[1], d["query"].shape[2] + 8, dtype=d["query"].dtype, device=dev)
        big[..., :-8] = d["query"]
        bt = torch.full((len(c["context_lens"]) + 2, c["block_tables"].shape[1] + 5), 7, dtype=torch.int32, device=dev)
        bt[:-2, :-5] = d["block_tables"]
        turned = dict(d, query=big[..., :-8], block_tables=bt[:-2, :-5], context_lens=d["context_lens"].int(),
                      weights=d["weights"].clone())
        if c["cu_seqlens_q"] is not None:
            turned["cu_seqlens_q"] = d["cu_seqlens_q"].long()
        assert torch.equal(mkv.paged_attention_weights(**turned), want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = mkv.paged_attention_weights(**dict(d, weights=d["weights"].clone()))
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
    ds, graphs = [on(dev, c) for c in cases], []
    for d in ds:
        mkv.paged_attention_weights(**d)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with graph_capture(graph):
            mkv.paged_attention_weights(**d)
        graphs.append(graph)
    g = torch.Generator(device=dev).manual_seed(1)
    for turn in range(4):
        befores = []
        for d in ds:
            d["query"].copy_(torch.randn(d["query"].shape, generator=g, device=dev))
            befores.append(d["weights"].clone())
        for graph in graphs:
            graph.replay()
        for d, before in zip(ds, befores):
            want = mkv.paged_attention_weights(**dict(d, weights=before))
            torch.cuda.synchronize()
            assert torch.equal(d["weights"], want), f"replay {turn}"


def test_nothing_to_do(dev):
    announce("weights: no sequences, no rows, empty contexts")
    c = on(dev, make("bf16", None, [20], 4, 2, 128, 16, seed=16))
    before = c["weights"].clone()
    none = dict(c, query=c["query"][:0], context_lens=c["context_lens"][:0], block_tables=c["block_tables"][:0])
    assert torch.equal(mkv.paged_attention_weights(**none), before)
    assert torch.equal(mkv.paged_attention_weights(**dict(c, block_tables=c["block_tables"][:, :0])), before)
    zero = dict(c, context_lens=torch.zeros_like(c["context_lens"]))
    assert torch.equal(mkv.paged_attention_weights(**zero), before)
    # a sequence without rows decays
    cu = torch.zeros(2, dtype=torch.int32, device=dev)
    got = mkv.paged_attention_weights(**dict(c, query=c["query"][:0], cu_seqlens_q=cu), decay=0.5)
    want, _ = oracle({n: v.cpu() if isinstance(v, torch.Tensor) else v
                      for n, v in dict(c, weights=before, query=c["query"][:0], cu_seqlens_q=cu).items()}, 0.5)
    assert torch.equal(got.cpu().double(), want)
