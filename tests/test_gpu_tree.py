"""GPU parity of tree attention (drafted tokens over the paged cache) against
its definition in float64.

Bounds.  An output is sum_j p_j v_j / sum_j p_j, so a relative error d of every
p moves it by at most d max|v|.  Rounding P to fp16 (fp16 and 1-byte caches):
2^-11.  bf16 caches carry P in two bf16 terms: 2^-8 of 2^-8.  The rest is fp32:
a score is a sum of 128 products (128 x 2^-24 of sum |q k| scale, below 16 here:
2^-13 in the exponent), the output and the normaliser are sums of up to 4096
terms (2^-12 at the very most, roundings being of both signs far less).  Together
below 2^-11 max|v| beside P's term, and the store's half step."""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce, assert_close_out
from mkv import workloads as W
from mkv.decode_state import graph_capture

pytestmark = pytest.mark.gpu

CACHES = {"fp32": (torch.float32, torch.float32, "auto"), "bf16": (torch.bfloat16, torch.bfloat16, "auto"),
          "fp16": (torch.float16, torch.float16, "auto"), "fp8": (torch.float8_e4m3fn, torch.bfloat16, "fp8_per_tensor"),
          "fp8_q16": (torch.float8_e4m3fn, torch.float16, "fp8_per_tensor"),
          "fp8_token": (torch.float8_e4m3fn, torch.bfloat16, "fp8_per_token_head"),
          "int8_token": (torch.int8, torch.float16, "int8_per_token_head")}
P_EPS = {"fp32": 0.0, "bf16": 2.0 ** -16}  # 2^-11 otherwise


def make(fmt, draft, prefix, Hq, Hkv, D, bs, seed=0, extra_rows=0, width=None, spread=1.0):
    """Inputs of one call on the CPU (random masks: any subset, with the row
    itself mostly among it), lists of drafted and prefix lengths."""
    g = torch.Generator().manual_seed(seed)
    cdt, qdt, mode = CACHES[fmt]
    B, total = len(draft), sum(draft) + extra_rows
    ctx = torch.tensor([d + p for d, p in zip(draft, prefix)], dtype=torch.int64)
    blocks = sum(-(-int(c) // bs) for c in ctx) + 3
    bt = W.fragmented_block_tables(ctx, bs, blocks, g)
    kv = [torch.randn(blocks, bs, Hkv, D, generator=g) for _ in range(2)]
    ks = vs = None
    if mode == "fp8_per_tensor":
        ks, vs = torch.tensor([0.013]), torch.tensor([0.011])
        kv = [(x / s).clamp(-448, 448) for x, s in zip(kv, (ks, vs))]
    elif mode != "auto":
        top = 127.0 if cdt == torch.int8 else 448.0
        ks, vs = ((torch.rand(blocks, bs, Hkv, generator=g) + 0.5) * 3 / top for _ in range(2))
        kv = [(x * top / 3).clamp(-top, top) for x in kv]
        if cdt == torch.int8:
            kv = [x.round() for x in kv]
    k, v = (x.to(cdt) for x in kv)
    q = (torch.randn(total, Hq, D, generator=g) * spread).to(qdt)
    cu = torch.tensor([0] + draft, dtype=torch.int32).cumsum(0).to(torch.int32)
    mask = torch.rand(total, width or max(draft + [1]), generator=g) < 0.5
    for s in range(B):
        for i in range(draft[s]):
            if i < mask.shape[1] and i % 5 != 3:
                mask[cu[s] + i, i] = True
    return dict(q=q, k=k, v=v, bt=bt, ctx=ctx, cu=cu, mask=mask, scale=1 / math.sqrt(D), Hq=Hq, Hkv=Hkv, D=D, bs=bs,
                ks=ks, vs=vs, mode=mode, fmt=fmt)


def dequantised(x, scale, mode):
    y = x.double()
    if scale is None:
        return y
    return y * (scale.double() if mode == "fp8_per_tensor" else scale.double()[..., None])


def reference(c):
    """Row by row, from the definition, in float64."""
    q, cu, ctx, bt, mask = c["q"].double(), c["cu"].tolist(), c["ctx"].tolist(), c["bt"], c["mask"]
    k, v = dequantised(c["k"], c["ks"], c["mode"]), dequantised(c["v"], c["vs"], c["mode"])
    out = torch.zeros_like(q)
    G = c["Hq"] // c["Hkv"]
    for s in range(len(ctx)):
        n = cu[s + 1] - cu[s]
        pos = torch.arange(ctx[s])
        page = bt[s, pos // c["bs"]].long()
        keys, vals = (x[page.clamp(min=0), pos % c["bs"]] for x in (k, v))
        first = max(ctx[s] - n, 0)
        for i in range(min(n, mask.shape[1])):
            sees = page >= 0
            for t in range(first, ctx[s]):
                j = t - first
                sees[t] &= bool(mask[cu[s] + i, j]) if j < mask.shape[1] else False
            if not bool(sees.any()):
                continue
            for h in range(c["Hq"]):
                score = keys[sees, h // G] @ q[cu[s] + i, h] * c["scale"]
                out[cu[s] + i, h] = torch.softmax(score, 0) @ vals[sees, h // G]
    return out


def run(c, dev, **over):
    t = {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in {**c, **over}.items()}
    return mkv.paged_attention_tree(t["q"], t["k"], t["v"], t["bt"], t["ctx"], t["cu"], t["mask"], t["scale"], t["Hq"],
                                    t["Hkv"], t["D"], t["bs"], k_scale=t["ks"], v_scale=t["vs"],
                                    kv_cache_dtype=t["mode"], out=t.get("out"))


def bound(c):
    top = float(dequantised(c["v"], c["vs"], c["mode"]).abs().max())
    return top * (P_EPS.get(c["fmt"], 2.0 ** -11) + 2.0 ** -11)


def check(c, dev, **over):
    got = run(c, dev, **over)
    total = int(c["cu"][-1])
    assert_close_out(got[:total], reference(c)[:total], c["q"].dtype, bound(c))
    return got


# (drafted, prefix, Hq, Hkv, D, bs)
SHAPES = {
    "one": ([1], [0], 2, 1, 128, 16),
    "pair": ([1, 2], [15, 0], 16, 8, 128, 16),
    "odd_group": ([5, 33, 1], [30, 200, 7], 12, 4, 128, 16),
    "rows32": ([16, 16], [300, 65], 16, 8, 128, 256),
    "rows64": ([17, 32, 3], [129, 31, 400], 8, 4, 128, 32),
    "rows128": ([40, 64], [500, 64], 4, 2, 128, 64),
    "rows256": ([64, 61, 2], [130, 1, 700], 8, 2, 128, 16),
    "two_blocks": ([70, 3], [90, 40], 16, 4, 128, 16),
    "group16": ([7, 20], [100, 33], 16, 1, 128, 16),
    "long": ([9], [3100], 2, 1, 128, 16),
    "d64": ([9, 24, 1], [70, 130, 3], 8, 4, 64, 16),
    "d64_group8": ([6, 17], [33, 260], 16, 2, 64, 32),
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("fmt", CACHES)
def test_against_the_definition(dev, fmt, shape):
    announce(f"tree {fmt} {shape}")
    check(make(fmt, *SHAPES[shape], seed=len(shape)), dev)


@pytest.mark.parametrize("fmt", ["bf16", "fp32", "fp8"])
def test_masks_lengths_and_padding(dev, fmt):
    """A batch as a captured step pads it: an inactive row (context 0), a
    sequence without drafted tokens, rows that see nothing at all (no prefix, an
    empty mask row), an absent block, a mask narrower than a tree, rows behind
    the last sequence."""
    announce(f"tree padding {fmt}")
    c = make(fmt, [4, 0, 3, 20, 6], [0, 40, 50, 33, 0], 8, 4, 128, 16, seed=3, extra_rows=5, width=16)
    c["ctx"][4] = 0       # padded: six rows, no keys
    c["mask"][0] = False  # sees nothing
    c["mask"][2] = False
    c["mask"][8] = False  # sees the prefix only
    c["bt"][2, 1] = -1
    want = reference(c)
    assert not bool(want[0].any()) and bool(want[8].any())
    out = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype, device=dev)
    got = check(c, dev, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((got[33:] == 7.0).all())           # behind the last sequence
    assert not bool(got[7 + 16:7 + 20].any())      # past the mask's width
    assert not bool(got[27:33].any()) and not bool(got[0].any())
    got = run(c, dev, ctx=c["ctx"].to(torch.int32))
    assert torch.equal(got[:33], out[:33])


@pytest.mark.parametrize("fmt", ["bf16", "fp16", "fp32", "fp8", "fp8_token", "int8_token"])
def test_values_that_are_not_finite_stay_where_they_are_seen(dev, fmt):
    """Slots behind the context and drafted tokens that a row does not see may
    hold anything; those that see an infinite or NaN value have it."""
    announce(f"tree not finite {fmt}")
    c = make(fmt, [6, 3], [37, 18], 8, 4, 128, 16, seed=5)
    clean = reference(c)
    c["mask"][:6, 2] = torch.tensor([False, True, True, False, True, False])
    c["mask"][:6, 4] = torch.tensor([False, False, True, False, True, True])
    page, row = int(c["bt"][0, 39 // 16]), 39 % 16
    page4, row4 = int(c["bt"][0, 41 // 16]), 41 % 16
    nan, inf = math.nan, math.inf
    dt = c["k"].dtype
    behind = int(c["bt"][1, 21 // 16]), 21 % 16  # the second context ends at 21
    if dt == torch.int8:
        for s in (c["ks"], c["vs"]):
            s[page, row] = nan
            s[behind] = inf
        c["vs"][page4, row4, 1] = inf
    else:
        c["k"][behind], c["v"][behind] = nan, nan
        c["k"][page, row, 0], c["v"][page, row] = nan, nan
        if dt != torch.float8_e4m3fn:
            c["v"][page4, row4, 2, 5], c["v"][page4, row4, 3, 7] = inf, -inf
        if c["mode"] == "fp8_per_token_head":
            c["vs"][page, row] = inf
            c["ks"][behind], c["vs"][behind] = nan, nan
    want = reference(c)
    assert bool(torch.isfinite(want[[0, 3]]).all()) and bool(want[1].isnan().any())
    got = run(c, dev).double().cpu()
    if c["mode"] in ("fp8_per_token_head", "int8_per_token_head"):
        # an infinite scale times a zero code is NaN in one arithmetic, infinite
        # in another: both are where the row sees the token
        assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    else:
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[got.isinf()], want[want.isinf()]) and torch.equal(got.isinf(), want.isinf())
    fine = torch.isfinite(want)
    top = float(clean.abs().max()) * 4
    assert float((got - want)[fine].abs().max()) <= top * 2.0 ** -7


def test_a_chain_is_decode(dev):
    """A tree that is a chain gives what decode gives token by token."""
    announce("tree chain")
    c = make("bf16", [5], [300], 16, 8, 128, 16, seed=9)
    c["mask"] = torch.ones(5, 5, dtype=torch.bool).tril()
    got = run(c, dev).float()
    for i in range(5):
        want = mkv.paged_attention_decode(c["q"][i:i + 1].to(dev), c["k"].to(dev), c["v"].to(dev), c["bt"].to(dev),
                                          torch.tensor([301 + i], device=dev), c["scale"], 16, 8, 128, 16).float()
        # both within bound() of the exact value before their roundings (2^-8)
        assert float((got[i] - want[0]).abs().max()) <= 2 * bound(c) + 2.0 ** -7 * float(want.abs().max())


@pytest.mark.parametrize("scale", [0.0, -0.09, 1.5])
def test_scales(dev, scale):
    announce(f"tree scale {scale}")
    for fmt in ("bf16", "fp8", "fp32"):
        c = make(fmt, [6, 2], [50, 9], 4, 2, 128, 16, seed=2, spread=0.3)
        c["scale"] = scale
        got = run(c, dev)
        # scores up to 1.5 x 128 x |q k| / ... : the exponent's error grows with the
        # scale, 2^-13 per 1/sqrt(128) of it
        assert_close_out(got, reference(c), c["q"].dtype, bound(c) * (1 + abs(scale) * 12))


def test_strides_and_layouts(dev):
    announce("tree strides")
    c = make("bf16", [6, 9], [50, 9], 4, 2, 128, 16, seed=4)
    want = run(c, dev)
    wide = torch.zeros(20, 40, dtype=torch.uint8, device=dev)
    wide[:15, 3:12] = c["mask"].to(dev).to(torch.uint8) * 255
    tables = torch.full((4, 9), -1, dtype=torch.int32, device=dev)
    tables[:2, :c["bt"].shape[1]] = c["bt"].to(dev)
    q = torch.randn(15, 8, 128, device=dev, dtype=torch.bfloat16)
    q[:, ::2] = c["q"].to(dev)
    got = run(c, dev, mask=wide[:, 3:12], bt=tables, q=q[:, ::2], cu=c["cu"].long())
    assert torch.equal(got, want)
    assert torch.equal(run(c, dev, mask=c["mask"].to(dev).t().contiguous().t()), want)


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^31 elements, its last pages used."""
    announce("tree large pool")
    Hkv, D, bs, N = 8, 128, 256, 8200
    k = torch.zeros(N, bs, Hkv, D, dtype=torch.float8_e4m3fn, device=dev)
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    c = make("fp8", [7, 4], [300, 20], 16, 8, D, bs, seed=6)
    n = c["k"].shape[0]
    k[N - n:], v[N - n:] = c["k"].to(dev), c["v"].to(dev)
    bt = torch.where(c["bt"] >= 0, c["bt"] + N - n, -1)
    assert torch.equal(run(c, dev, k=k, v=v, bt=bt.to(torch.int32)), run(c, dev))


def test_captured_and_replayed(dev):
    """A captured call, replayed with other lengths and masks between eager
    calls; two graphs, replayed on two streams at once."""
    announce("tree graph")
    a, b = (make("bf16", [8, 8], [p, 700 - p], 16, 8, 128, 16, seed=p) for p in (40, 500))
    for c in (a, b):
        c["bt"] = torch.nn.functional.pad(c["bt"], (0, 64 - c["bt"].shape[1]), value=-1)
    want = [run(c, dev) for c in (a, b)]
    n = max(a["k"].shape[0], b["k"].shape[0])

    def state(c):
        s = {k: x.to(dev) if isinstance(x, torch.Tensor) else x for k, x in c.items()}
        s["k"], s["v"] = (torch.nn.functional.pad(x, (0,) * 7 + (n - x.shape[0],)) for x in (s["k"], s["v"]))
        return s

    live = [state(a), state(b)]
    outs, graphs = [torch.empty_like(s["q"]) for s in live], []
    for s, o in zip(live, outs):
        run(s, dev, out=o)
        g = torch.cuda.CUDAGraph()
        with graph_capture(g):
            run(s, dev, out=o)
        graphs.append(g)
    other = [state(b), state(a)]
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    for turn in range(4):
        for s, o, new in zip(live, outs, other if turn % 2 else [state(a), state(b)]):
            o.zero_()
            for k, x in new.items():
                if isinstance(x, torch.Tensor):
                    s[k].copy_(x)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        run(live[0], dev)
        torch.cuda.synchronize()
        for i, o in enumerate(outs):
            assert torch.equal(o, want[i ^ (turn % 2)]), f"replay {turn}, graph {i}"


def test_same_bits_every_time(dev):
    announce("tree determinism")
    c = make("fp8", [16, 9, 30], [900, 20, 3000], 16, 4, 128, 16, seed=8)
    want = run(c, dev)
    for _ in range(5):
        assert torch.equal(run(c, dev), want)


def test_attention_layer_runs_a_tree_step(dev):
    """mkv.Attention with a Context that carries a tree mask: appends the
    drafted tokens' K and V, then attends as the function does."""
    announce("tree layer")
    from mkv import context as C

    c = make("bf16", [5, 3], [40, 12], 8, 4, 128, 16, seed=11)
    layer = mkv.Attention(8, 128, num_kv_heads=4, block_size=16)
    layer.k_cache, layer.v_cache = c["k"].to(dev), c["v"].to(dev)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(8, 4, 128, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    slots = [int(c["bt"][s, p // 16]) * 16 + p % 16 for s, n, P in ((0, 5, 40), (1, 3, 12)) for p in range(P, P + n)]
    C.set_context(True, cu_seqlens_q=c["cu"].to(dev), slot_mapping=torch.tensor(slots, device=dev),
                  context_lens=c["ctx"].to(dev), block_tables=c["bt"].to(dev), tree_mask=c["mask"].to(dev))
    try:
        got = layer(c["q"].to(dev), k, v)
    finally:
        C.reset_context()
    flat = [x.view(-1, 4, 128) for x in (c["k"], c["v"])]
    for x, new in zip(flat, (k, v)):
        x[torch.tensor(slots)] = new.cpu()
    assert torch.equal(layer.k_cache.cpu(), c["k"])
    assert_close_out(got.view(8, 8, 128), reference(c), torch.bfloat16, bound(c))
