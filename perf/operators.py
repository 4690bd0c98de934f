"""The operators of a speculative or forked decode step, with their plain forms.

Operators (``op``):

* ``tree``     attention of trees of drafted tokens over a paged cache: row i of
               a sequence sees the cached prefix and the drafted tokens its mask
               row names
* ``logprobs`` log probabilities of given tokens, the entropy of each row's
               distribution and its top alternatives
* ``copy``     copies of whole pages in every layer's K and V pool
* ``fork``     page tables: rows continue other rows' sequences (sharing full
               pages, a copy of a part-filled last one), grow or are freed
* ``compact``  the accepted drafted tokens' cache rows moved up behind the prefix

Cache formats (``fmt``) of ``tree``: ``bf16``, ``fp16``, ``fp32``, ``fp8``
(per-tensor scales), ``fp8_token`` and ``int8_token`` (a scale per token and KV
head).  A case's lengths follow from its sizes alone; the seed decides their
order, the page tables and every value.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False
DEV = "cuda"
CACHE_DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
               "fp8": torch.float8_e4m3fn, "fp8_token": torch.float8_e4m3fn, "int8_token": torch.int8}
MODE = {"fp8": "fp8_per_tensor", "fp8_token": "fp8_per_token_head", "int8_token": "int8_per_token_head"}
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a lone request's verification step: eight drafted tokens
        dict(name="tree_b1", op="tree", fmt="bf16", batch=1, draft_lo=8, draft_hi=8, lo=700, hi=700,
             heads=16, kv_heads=8, head_dim=128, block=256),
        # the engine's decode batch, sixteen drafted tokens each, its cache format
        dict(name="tree_engine_fp8", op="tree", fmt="fp8", batch=60, draft_lo=16, draft_hi=16, lo=300, hi=800,
             heads=16, kv_heads=8, head_dim=128, block=256),
        # wide trees, four query heads to a KV head: the most arithmetic to a cached byte
        dict(name="tree_wide", op="tree", fmt="bf16", batch=8, draft_lo=64, draft_hi=64, lo=1024, hi=4096,
             heads=32, kv_heads=8, head_dim=128, block=256),
        # two long documents, ragged trees: the cache's bytes
        dict(name="tree_long", op="tree", fmt="bf16", batch=2, draft_lo=17, draft_hi=32, lo=98304, hi=131072,
             heads=32, kv_heads=8, head_dim=128, block=256),
        # the sampled tokens of one engine step
        dict(name="logprobs_step", op="logprobs", dtype="bf16", rows=60, vocab=151936, tokens=1, top=5, masked=0),
        # scoring a prompt
        dict(name="logprobs_prompt", op="logprobs", dtype="bf16", rows=1024, vocab=151936, tokens=1, top=20, masked=0),
        # copy-on-write of a few pages
        dict(name="copy_few", op="copy", dtype="bf16", layers=28, pages=256, block=16, kv_heads=8, head_dim=128, pairs=4),
        # a swap of many sequences' pages
        dict(name="copy_many", op="copy", dtype="bf16", layers=28, pages=1024, block=16, kv_heads=8, head_dim=128,
             pairs=320),
        # one prompt answered four times
        dict(name="fork_samples", op="fork", dtype="bf16", layers=28, rows=8, width=8, extra=8, block=256, kv_heads=8,
             head_dim=128, lo=700, hi=700, group=4, beams=0, freed=0, grow=1),
        # a beam step: every row of a group continues one of its beams
        dict(name="fork_beams", op="fork", dtype="bf16", layers=28, rows=64, width=64, extra=128, block=16, kv_heads=8,
             head_dim=128, lo=300, hi=800, group=4, beams=1, freed=0, grow=16),
        # one request's accepted path of four
        dict(name="compact_b1", op="compact", dtype="bf16", layers=28, batch=1, block=16, kv_heads=8, head_dim=128,
             lo=200, hi=200, draft=16, accepted=4),
        # the engine's batch, up to eight accepted of 64
        dict(name="compact_b60", op="compact", dtype="bf16", layers=28, batch=60, block=16, kv_heads=8, head_dim=128,
             lo=60, hi=240, draft=64, accepted=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "logprobs", "logprobs", "copy", "fork", "compact"])
    if op == "tree":
        while True:
            kv_heads = rng.choice([1, 2, 4, 8])
            hi = _log(rng, 1, 60000)
            d_hi = _log(rng, 1, 64)
            c = dict(op=op, fmt=rng.choice(list(CACHE_DTYPE)), batch=_log(rng, 1, 96), draft_lo=rng.randint(1, d_hi),
                     draft_hi=d_hi, lo=rng.randint(0, hi), hi=hi, heads=kv_heads * rng.choice([1, 2, 3, 4, 8]),
                     kv_heads=kv_heads, head_dim=128, block=rng.choice([16, 32, 256]))
            if kv_heads > 1 and rng.random() < 0.25:
                c["head_dim"] = 64
            w = work(c)
            if w["bytes"] < 5e8 and w["flops"] < (5e9 if c["fmt"] == "fp32" else 5e10):
                return c
    if op == "logprobs":
        rows, vocab = _log(rng, 1, 4096), _log(rng, 2, 262144)
        return dict(op=op, dtype=rng.choice(list(DTYPE)), rows=max(1, min(rows, 40_000_000 // vocab)), vocab=vocab,
                    tokens=rng.choice([1, 1, 4]), top=min(vocab, rng.choice([0, 1, 5, 20, 64])), masked=rng.choice([0, 1]))
    pool = dict(dtype=rng.choice(list(DTYPE)), layers=_log(rng, 1, 28), block=rng.choice([16, 32, 64]),
                kv_heads=rng.choice([1, 2, 8]), head_dim=rng.choice([64, 128]))
    if op == "copy":
        pages = _log(rng, 4, 256)
        return dict(op=op, pages=pages, pairs=rng.randint(1, pages // 2), **pool)
    hi = _log(rng, 1, 400)
    lo = rng.randint(1, hi)
    if op == "fork":
        group = rng.choice([1, 2, 4, 5])
        rows = group * _log(rng, 1, 16)
        width = hi // pool["block"] + 3
        return dict(op=op, rows=rows, width=width, extra=rows * 3, lo=lo, hi=hi, group=group, beams=rng.choice([0, 1]),
                    freed=rng.randint(0, rows // 4), grow=rng.choice([0, 1, 33]), **pool)
    draft = _log(rng, 1, 64)
    return dict(op=op, batch=_log(rng, 1, 64), lo=lo, hi=hi, draft=draft, accepted=rng.randint(1, min(12, draft)), **pool)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _page_tables(rng, counts, width, pages):
    """Each sequence's pages in random places, padded with -1."""
    ids = rng.sample(range(pages), sum(counts))
    rows, at = [], 0
    for n in counts:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return rows


def _tree_mask(rng, lens, width):
    """Rows of ancestors (and the token itself) of random trees, parents before
    children; a parent of -1 is the cached prefix's last token."""
    rows = []
    for n in lens:
        seen = []
        for i in range(n):
            parent = rng.randint(max(-1, i - 6), i - 1)
            seen.append((seen[parent] if parent >= 0 else 0) | (1 << i))
        rows += [[bool(s >> j & 1) for j in range(width)] for s in seen]
    return rows


def _pool(case, gen, pages):
    shape = (2 * case["layers"], pages, case["block"], case["kv_heads"], case["head_dim"])
    return torch.randn(shape, generator=gen, device=DEV, dtype=DTYPE[case["dtype"]])


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)

    def dev(x, dtype):
        return torch.tensor(x, dtype=dtype, device=DEV)

    if case["op"] == "tree":
        B, H, D, bs = case["batch"], case["kv_heads"], case["head_dim"], case["block"]
        lens, prefix = _spread(case["draft_lo"], case["draft_hi"], B), _spread(case["lo"], case["hi"], B)
        rng.shuffle(lens)
        ctx = [p + n for p, n in zip(prefix, lens)]
        counts = [-(-c // bs) for c in ctx]
        pages = sum(counts) + 3
        total, fmt = sum(lens), case["fmt"]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        shape = (pages, bs, H, D)
        kv = [torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32 if fmt == "fp32" else torch.bfloat16)
              for _ in range(2)]
        s.update(k_scale=None, v_scale=None)
        if fmt == "fp8":
            s.update(k_scale=dev([5.5 / 448], torch.float32), v_scale=dev([5.3 / 448], torch.float32))
            kv = [(x * (448 / 5.5)).clamp(-448, 448) for x in kv]
        elif fmt.endswith("_token"):
            top = 448 if fmt == "fp8_token" else 127
            s.update({n: (torch.rand(shape[:3], generator=gen, device=DEV) * 0.5 + 0.75) * (3 / top)
                      for n in ("k_scale", "v_scale")})
            kv = [(x * (top / 3)).clamp(-top, top) for x in kv]
        s["k_cache"], s["v_cache"] = (x.to(CACHE_DTYPE[fmt]) for x in kv)
        qt = DTYPE.get(fmt, torch.bfloat16)
        s["q"] = (torch.randn(total, case["heads"], D, generator=gen, device=DEV) * 1.5).to(qt)
        s["block_tables"] = dev(_page_tables(rng, counts, max(counts), pages), torch.int32)
        s["context_lens"], s["cu"] = dev(ctx, torch.int64), dev(cu, torch.int32)
        s["mask"] = dev(_tree_mask(rng, lens, case["draft_hi"]), torch.bool)
        s["scale"] = 1 / math.sqrt(D)
    elif case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        x = (torch.randn(R, V, generator=gen, device=DEV) * 3).to(DTYPE[case["dtype"]])
        if case["masked"]:  # a grammar that leaves about a third of the vocabulary
            x.masked_fill_(torch.rand(V, generator=gen, device=DEV) < 0.66, -math.inf)
            x[:, V // 2] = 0.5
        s["logits"] = x
        s["tokens"] = torch.randint(V, (R, case["tokens"]), generator=gen, device=DEV)
        if case["masked"]:
            s["tokens"][:, 0] = V // 2
    elif case["op"] == "copy":
        ids = rng.sample(range(case["pages"]), 2 * case["pairs"])
        s["pool"] = _pool(case, gen, case["pages"])
        s["src"], s["dst"] = (dev(x, torch.int64) for x in (ids[::2], ids[1::2]))
    elif case["op"] == "fork":
        R, W, bs, group = case["rows"], case["width"], case["block"], case["group"]
        lens = _spread(case["lo"], case["hi"], R)
        rng.shuffle(lens)
        held = [-(-n // bs) for n in lens]
        pages = sum(held) + case["extra"]
        tables = _page_tables(rng, held, W, pages)
        refs = [0] * pages
        for row in tables:
            for p in row:
                if p >= 0:
                    refs[p] = 1
        # samples continue their group's first row, beams any row of it
        parents = [i - i % group + (rng.randrange(group) if case["beams"] and i % group else 0) for i in range(R)]
        for i in rng.sample(range(R), case["freed"]):
            parents[i] = -1
        s["pool"] = _pool(case, gen, pages)
        s["block_tables"] = dev([[max(p, 0) for p in row] for row in tables], torch.int32)
        s["seq_lens"], s["held"] = dev(lens, torch.int64), dev(held, torch.int32)
        s["ref_counts"], s["parents"] = dev(refs, torch.int32), dev(parents, torch.int64)
        s["tokens"] = dev([0 if p < 0 else lens[p] + case["grow"] for p in parents], torch.int64)
    else:
        B, bs, n = case["batch"], case["block"], case["draft"]
        prefix = _spread(case["lo"], case["hi"], B)
        rng.shuffle(prefix)
        counts = [-(-(p + n) // bs) for p in prefix]
        accepted = []
        for _ in range(B):
            k = rng.randint(1, case["accepted"])
            accepted.append(sorted(rng.sample(range(n), k)) + [-1] * (case["accepted"] - k))
        s["pool"] = _pool(case, gen, sum(counts))
        s["block_tables"] = dev(_page_tables(rng, counts, max(counts), sum(counts)), torch.int32)
        s["prefix"], s["accepted"] = dev(prefix, torch.int64), dev(accepted, torch.int64)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _mkv():
    root = str(Path(__file__).resolve().parent.parent / "mini-kvllm_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mkv

    return mkv


def run(state):
    return _RUN[state["case"]["op"]](state)


def _dequantised(cache, scale):
    x = cache.float()
    if scale is None:
        return x
    return x * (scale if scale.numel() == 1 else scale[..., None])


def _tree(s):
    c = s["case"]
    H, D, bs = c["kv_heads"], c["head_dim"], c["block"]
    if own:
        return _mkv().paged_attention_tree(
            s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["context_lens"], s["cu"], s["mask"], s["scale"],
            c["heads"], H, D, bs, k_scale=s["k_scale"], v_scale=s["v_scale"], kv_cache_dtype=MODE.get(c["fmt"], "auto"))
    q, cu, ctx, mask = s["q"].float(), s["cu"].long(), s["context_lens"], s["mask"]
    B, W = s["block_tables"].shape
    G, M, L = c["heads"] // H, mask.shape[1], W * bs
    pages = s["block_tables"].long().clamp(min=0)
    k, v = (_dequantised(s[n + "_cache"][pages], s[n + "_scale"] if c["fmt"] == "fp8" or s[n + "_scale"] is None
                         else s[n + "_scale"][pages]).reshape(B, L, H, D).transpose(1, 2) for n in ("k", "v"))
    # sequences padded to the widest tree
    rows = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu, rows, right=True) - 1
    at = seq * M + rows - cu[seq]
    qp = q.new_zeros(B * M, H * G * D).index_copy_(0, at, q.reshape(-1, H * G * D))
    qp = qp.reshape(B, M, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * M, D)
    tree = torch.zeros(B * M, M, dtype=torch.bool, device=q.device).index_copy_(0, at, mask).reshape(B, M, M)
    pos = torch.arange(L, device=q.device)
    prefix = (ctx - (cu[1:] - cu[:-1]))[:, None]
    col = (pos - prefix).clamp(0, M - 1)
    sees = (pos < prefix)[:, None, :] | (tree.gather(2, col[:, None, :].expand(B, M, L))
                                         & ((pos >= prefix) & (pos < ctx[:, None]))[:, None, :])
    score = (qp @ k.transpose(2, 3)).reshape(B, H, G, M, L) * s["scale"]
    score = score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.reshape(B, H, G * M, L) @ v).reshape(B, H, G, M, D) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(B * M, H * G, D)[at].to(s["q"].dtype)


def _logprobs(s):
    if own:
        r = _mkv().token_logprobs(s["logits"], s["tokens"], s["case"]["top"])
        return r.logprobs, r.entropy, r.top_logprobs, r.top_indices
    x = s["logits"].float()
    y = x - x.amax(-1, keepdim=True)
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = (log_total - torch.where(e > 0, e * y, 0).sum(-1, keepdim=True) / total)[:, 0]
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["case"]["top"]]
    return y.gather(1, s["tokens"]) - log_total, entropy, y.gather(1, order) - log_total, order


def _pages_of(s):
    """The handle on every layer's pools that a program keeps."""
    if "pages" not in s:
        s["pages"] = _mkv().CachePages(list(s["pool"].unbind(0)))
    return s["pages"]


def _copy(s):
    if own:
        _pages_of(s).copy(s["src"], s["dst"])
    else:
        s["pool"][:, s["dst"]] = s["pool"][:, s["src"]]
    return s["pool"]


def _fork(s):
    if own:
        if "pages" not in s:
            s["pages"] = _mkv().PagePool(s["block_tables"], s["seq_lens"], _mkv().CachePages(list(s["pool"].unbind(0))),
                                         ref_counts=s["ref_counts"], held=s["held"])
        granted = s["pages"].assign(s["parents"], s["tokens"])
    else:
        granted = _assign(s, s["block_tables"], s["seq_lens"], s["held"], s["ref_counts"], s["parents"], s["tokens"])
    return [s[n] for n in ("block_tables", "seq_lens", "held", "ref_counts")] + [granted, s["pool"]]


def _assign(s, tables, lens, held, refs, parents, tokens):
    bs = s["case"]["block"]
    R, W = tables.shape
    rows, cols = (torch.arange(n, device=tables.device) for n in (R, W))
    src, stays, gone = parents.clamp(min=0), parents == rows, parents < 0
    # the pages each row keeps of its parent's
    keep = torch.where(gone, 0, torch.where(stays, held, (lens[src] + bs - 1).div(bs, rounding_mode="floor")))
    new_lens = torch.where(gone, 0, lens[src])
    new = torch.where(cols < keep[:, None], tables[src], 0)
    refs += torch.bincount(new[cols < keep[:, None]], minlength=refs.numel()).to(refs.dtype)
    refs -= torch.bincount(tables[cols < held[:, None]], minlength=refs.numel()).to(refs.dtype)
    # a part-filled last page that others hold too is copied; its first row keeps it
    fill = new_lens % bs
    at = (new_lens // bs).clamp(max=W - 1)
    last = torch.where(fill > 0, new.gather(1, at[:, None])[:, 0].long(), -1 - rows)
    alike = last[:, None] == last
    count = refs[last.clamp(min=0)]
    first = (alike & (rows[:, None] > rows)).sum(1) == 0
    copies = (fill > 0) & (count > 1) & ~(first & (count == alike.sum(1)))
    want = (tokens + bs - 1).div(bs, rounding_mode="floor")
    fits = gone & (tokens <= 0) | (want <= W)
    grow = (want - keep).clamp(min=0)
    need = torch.where(fits, copies + grow, 0)
    spare = (refs == 0).nonzero()[:, 0]
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= spare.numel()))
    # a row that was refused is freed, or stays as it was
    freed = ~granted & ~stays
    dropped = freed[:, None] & (cols < keep[:, None])
    refs -= torch.bincount(new[dropped], minlength=refs.numel()).to(refs.dtype)
    new, new_lens, keep = (torch.where(m, 0, x) for m, x in ((freed[:, None], new), (freed, new_lens), (freed, keep)))
    grow, copies = grow * granted, copies & granted
    start = upto - need
    page = spare[(start[:, None] + copies[:, None] + cols - keep[:, None]).clamp(0, max(spare.numel() - 1, 0))] \
        if spare.numel() else new
    grown = (cols >= keep[:, None]) & (cols < (keep + grow)[:, None])
    new = torch.where(grown, page.to(new.dtype), new)
    refs += torch.bincount(new[grown], minlength=refs.numel()).to(refs.dtype)
    which = copies.nonzero()[:, 0]
    if which.numel():
        old, fresh = last[which], spare[start[which]]
        new[which, at[which]] = fresh.to(new.dtype)
        refs += torch.bincount(fresh, minlength=refs.numel()).to(refs.dtype)
        refs -= torch.bincount(old, minlength=refs.numel()).to(refs.dtype)
        live = (torch.arange(bs, device=tables.device) < fill[which][:, None])[None, :, :, None, None]
        s["pool"][:, fresh] = torch.where(live, s["pool"][:, old], s["pool"][:, fresh])
    tables.copy_(new)
    lens.copy_(new_lens)
    held.copy_(keep + grow)
    return granted


def _compact(s):
    if own:
        _pages_of(s).compact(s["block_tables"], s["prefix"], s["accepted"])
        return s["pool"]
    bs, accepted, prefix, pool = s["case"]["block"], s["accepted"], s["prefix"][:, None], s["pool"]
    src = prefix + accepted.clamp(min=0)
    dst = prefix + torch.arange(accepted.shape[1], device=accepted.device)
    tables = s["block_tables"].long()
    src, dst = (tables.gather(1, p // bs) * bs + p % bs for p in (src, dst))
    moved = accepted >= 0
    rows = pool.view(pool.shape[0], -1, pool.shape[3] * pool.shape[4])
    rows[:, dst[moved]] = rows[:, src[moved]]
    return pool


_RUN = {"tree": _tree, "logprobs": _logprobs, "copy": _copy, "fork": _fork, "compact": _compact}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "tree":
        lens = _spread(c["draft_lo"], c["draft_hi"], c["batch"])
        n, prefix = sum(lens), sum(_spread(c["lo"], c["hi"], c["batch"]))
        size = torch.empty(0, dtype=CACHE_DTYPE[c["fmt"]]).element_size()
        q_size = 4 if c["fmt"] == "fp32" else 2
        per_token = c["kv_heads"] * (c["head_dim"] * size + (4 if c["fmt"].endswith("_token") else 0)) * 2
        pairs = prefix * n / c["batch"] + sum(x * (x + 1) / 2 for x in lens)
        return dict(bytes=(prefix + n) * per_token + 2 * n * c["heads"] * c["head_dim"] * q_size + n * c["draft_hi"],
                    flops=4 * pairs * c["heads"] * c["head_dim"])
    if c["op"] == "logprobs":
        size = 4 if c["dtype"] == "fp32" else 2
        return dict(bytes=c["rows"] * (c["vocab"] * size + 12 * c["tokens"] + 4 + 12 * c["top"]),
                    flops=c["rows"] * c["vocab"] * 4)
    row = 2 * c["layers"] * c["kv_heads"] * c["head_dim"] * (4 if c["dtype"] == "fp32" else 2)
    if c["op"] == "copy":
        return dict(bytes=2 * c["pairs"] * (c["block"] * row + 8), flops=0)
    if c["op"] == "fork":
        lens = _spread(c["lo"], c["hi"], c["rows"])
        g = c["group"]
        parents = 1 + (g - 1) * (1 - (1 - 1 / g) ** (g - 1)) if c["beams"] else 1  # a group's rows that are continued
        share = (c["rows"] - c["freed"]) / c["rows"] * (1 - parents / g)  # rows that need a copy of a page
        return dict(bytes=2 * share * row * sum(n % c["block"] for n in lens) + 8 * c["rows"] * (c["width"] + 5), flops=0)
    return dict(bytes=2 * c["batch"] * (c["accepted"] + 1) / 2 * row + 8 * c["batch"] * (c["accepted"] + 2), flops=0)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    bs = case.get("block")
    if case["op"] == "tree":
        out, G = [], case["heads"] // case["kv_heads"]
        cu, ctx, tables = s["cu"].tolist(), s["context_lens"].tolist(), s["block_tables"].tolist()
        for b in range(case["batch"]):
            n = cu[b + 1] - cu[b]
            ids = torch.tensor(tables[b][:-(-ctx[b] // bs)], device=DEV)
            kv = []
            for name in ("k", "v"):
                x = s[name + "_cache"][ids].double()
                if s[name + "_scale"] is not None:
                    x = x * (s[name + "_scale"].double() if case["fmt"] == "fp8" else s[name + "_scale"][ids].double()[..., None])
                kv.append(x.flatten(0, 1)[:ctx[b]])
            hidden = torch.zeros(n, ctx[b], dtype=torch.bool, device=DEV)
            hidden[:, ctx[b] - n:] = ~s["mask"][cu[b]:cu[b + 1], :n]
            heads = []
            for h in range(case["heads"]):
                score = s["q"][cu[b]:cu[b + 1], h].double() @ kv[0][:, h // G].t().contiguous() * s["scale"]
                heads.append(torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ kv[1][:, h // G].contiguous())
            out.append(torch.stack(heads, 1))
        return torch.cat(out)
    if case["op"] == "logprobs":
        lp, ent, top = [], [], []
        for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
            x = torch.log_softmax(x.double(), -1)
            lp.append(x.gather(1, t))
            ent.append(-torch.where(x > -math.inf, x.exp() * x, 0).sum(-1))
            top.append(torch.topk(x, case["top"], -1).values)
        return torch.cat(lp), torch.cat(ent), torch.cat(top), None
    pool = s["pool"].double()
    if case["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pool[:, b] = pool[:, a]
        return pool
    tables = s["block_tables"].tolist()
    if case["op"] == "compact":
        slots = pool.flatten(1, 2)
        for row, p, idx in zip(tables, s["prefix"].tolist(), s["accepted"].tolist()):
            for j, i in enumerate(idx):
                if i >= 0:  # in rising order: a row is read before it is written over
                    a, b = p + i, p + j
                    slots[:, row[b // bs] * bs + b % bs] = slots[:, row[a // bs] * bs + a % bs]
        return pool
    lens, held, parents = s["seq_lens"].tolist(), s["held"].tolist(), s["parents"].tolist()
    new = [[] if p < 0 else tables[p][:held[p] if p == i else -(-lens[p] // bs)] for i, p in enumerate(parents)]
    holders = {}
    for i, row in enumerate(new):
        for page in row:
            holders.setdefault(page, []).append(i)
    spare = (page for page in range(pool.shape[1]) if page not in holders)
    for i, (row, p, t) in enumerate(zip(new, parents, s["tokens"].tolist())):
        fill = lens[p] % bs if p >= 0 else 0
        old = row[lens[p] // bs] if fill else -1
        if fill and holders[old][0] != i:
            fresh = next(spare)
            pool[:, fresh, :fill] = pool[:, old, :fill]
        for _ in range(-(-t // bs) - len(row)):
            next(spare)
    return [None] * 5 + [pool]
