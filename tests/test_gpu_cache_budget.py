"""GPU tests of the operators that decide what stays in the cache, together, as a
program uses them.

* Sequences that grow, are cut to a budget and give pages back, their drafted tokens
  verified and compacted, against lists of keys, values and weights per layer and head
  in float64 on the CPU.
* The attention layer and the engine accumulate weights: what every row gives away sums
  to one a query head, and the tokens generated are the same.
"""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce
from mkv import context as C
from mkv import engine as E

pytestmark = pytest.mark.gpu

L, HQ, H, D, BS = 2, 4, 2, 128, 16
G = HQ // H


class Lists:
    """One layer's tokens of one sequence: [head] -> keys, values, weights."""

    def __init__(self):
        self.k, self.v, self.w = ([[] for _ in range(H)] for _ in range(3))

    def append(self, k, v):
        for h in range(H):
            self.k[h].append(k[h].double())
            self.v[h].append(v[h].double())
            self.w[h].append(0.0)

    def attend(self, q, rows, decay):
        """Outputs of the last `rows` tokens' queries (rows, HQ, D), weights taken."""
        n = len(self.k[0])
        out = torch.zeros(rows, HQ, D, dtype=torch.float64)
        for h in range(H):
            k, v = torch.stack(self.k[h]), torch.stack(self.v[h])
            add = torch.zeros(n, dtype=torch.float64)
            for j in range(G):
                s = q[:, h * G + j].double() @ k.t() / math.sqrt(D)
                hidden = torch.arange(n)[None] > torch.arange(n - rows, n)[:, None]
                p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                out[:, h * G + j] = p @ v
                add += p.sum(0)
            self.w[h] = [(decay * w if i < n - rows else 0.0) + float(a) for i, (w, a) in enumerate(zip(self.w[h], add))]
        return out

    def choose(self, budget, sinks, recent):
        """Kept tokens by head, and the smallest gap to what is left out."""
        n, kept, gap = len(self.k[0]), [], math.inf
        for h in range(H):
            mid = sorted(range(sinks, n - recent), key=lambda i: (-self.w[h][i], i))
            m = budget - sinks - recent
            if 0 < m < len(mid):
                a, b = self.w[h][mid[m - 1]], self.w[h][mid[m]]
                gap = min(gap, (a - b) / max(a, 1e-30))
            kept.append(list(range(sinks)) + sorted(mid[:m]) + list(range(n - recent, n)))
        return kept, gap

    def keep(self, kept):
        for xs in (self.k, self.v, self.w):
            for h in range(H):
                xs[h] = [xs[h][i] for i in kept[h]]


def test_sequences_within_a_budget_decode_and_verify(dev):
    announce("cache budget: weights, eviction, trim, drafts verified and compacted, fp32")
    g = torch.Generator().manual_seed(31)
    pages, rows_max, width, budget, sinks, recent = 40, 3, 10, 40, 2, 8
    k_caches = [torch.zeros(pages, BS, H, D, device=dev) for _ in range(L)]
    v_caches = [torch.zeros(pages, BS, H, D, device=dev) for _ in range(L)]
    weights = [torch.full((pages, BS, H), math.nan, device=dev) for _ in range(L)]
    eviction = mkv.CacheEviction(k_caches, v_caches, weights)
    tables = torch.zeros(rows_max, width, dtype=torch.int32, device=dev)
    lens = torch.zeros(rows_max, dtype=torch.int64, device=dev)
    pool = mkv.PagePool(tables, lens, mkv.CachePages(k_caches + v_caches + weights))
    lists = [[Lists() for _ in range(rows_max)] for _ in range(L)]
    stay = torch.arange(rows_max, device=dev)

    def t(x, dtype=torch.int64):
        return torch.tensor(x, dtype=dtype, device=dev)

    def step(new, decay=0.9, accumulate=True):
        """New tokens of every row through both layers; outputs against the lists."""
        before = lens.tolist()
        ends = [a + n for a, n in zip(before, new)]
        assert pool.assign(stay, t(ends)).tolist() == [True] * rows_max
        row = torch.tensor([r for r, n in enumerate(new) for _ in range(n)])
        pos = torch.tensor([a + i for a, n in zip(before, new) for i in range(n)])
        slots = tables[row.to(dev), (pos // BS).to(dev)].long() * BS + (pos % BS).to(dev)
        cu = torch.tensor([0] + new).cumsum(0)
        lens.copy_(t(ends))
        for i in range(L):
            k, v = (torch.randn(len(row), H, D, generator=g) for _ in range(2))
            q = torch.randn(len(row), HQ, D, generator=g) * 2
            mkv.store_kvcache(k.to(dev), v.to(dev), k_caches[i], v_caches[i], slots, BS)
            qd = q.to(dev)
            if max(new) == 1:
                o = mkv.paged_attention_decode(qd, k_caches[i], v_caches[i], tables, lens, 1 / math.sqrt(D), HQ, H, D, BS)
                kw = {}
            else:
                o = mkv.paged_attention_prefill_triton(qd, k_caches[i], v_caches[i], tables, lens, cu.int().to(dev),
                                                       pos.to(dev), 1 / math.sqrt(D), HQ, H, D, BS)
                kw = dict(cu_seqlens_q=cu.int().to(dev))
            mkv.paged_attention_weights(qd, k_caches[i], weights[i], tables, lens, 1 / math.sqrt(D), HQ, H, D, BS,
                                        decay=decay, **kw)
            for r, n in enumerate(new):
                if n == 0:
                    continue
                for x in range(cu[r], cu[r + 1]):
                    lists[i][r].append(k[x], v[x])
                want = lists[i][r].attend(q[cu[r]:cu[r + 1]], n, decay)
                assert float((o[cu[r]:cu[r + 1]].cpu().double() - want).abs().max()) <= 2e-3

    def compare():
        for i in range(L):
            for r in range(rows_max):
                for h in range(H):
                    n = len(lists[i][r].w[h])
                    j = torch.arange(n)
                    s = tables[r].cpu()[j // BS].long() * BS + j % BS
                    got = weights[i].flatten(0, 1)[s.to(dev), h].cpu().double()
                    want = torch.tensor(lists[i][r].w[h], dtype=torch.float64)
                    assert float((got - want).abs().max()) <= 1e-3 * max(1.0, float(want.max()))
                    keys = k_caches[i].flatten(0, 1)[s.to(dev), h].cpu().double()
                    assert torch.equal(keys, torch.stack(lists[i][r].k[h]))

    def evict():
        n = lens.tolist()
        choices = [[lists[i][r].choose(budget, sinks, recent) if n[r] > budget else None for r in range(rows_max)]
                   for i in range(L)]
        lens.copy_(eviction.evict(tables, lens, budget, sinks=sinks, recent=recent))
        pool.trim()
        assert lens.tolist() == [min(x, budget) for x in n]
        for i in range(L):
            for r in range(rows_max):
                if choices[i][r] is not None:
                    assert choices[i][r][1] > 1e-5, "an input on the border says nothing"
                    lists[i][r].keep(choices[i][r][0])
        held = pool.held.tolist()
        assert held == [-(-x // BS) for x in lens.tolist()] and sum(pool.ref_counts.tolist()) == sum(held)

    step([90, 30, 61])
    compare()
    evict()
    compare()
    for turn in range(14):
        step([1, 1, 1])
        if turn % 5 == 4:
            evict()
    compare()
    evict()
    # drafted chains behind it: root and three drafted tokens a row, accepted ones kept
    V, n = 50, 4
    before = lens.tolist()
    step([n] * rows_max)
    target, draft = torch.randn(rows_max * n, V, generator=g), torch.randn(rows_max * n, V, generator=g)
    ids = torch.randint(0, V, (rows_max * n,), generator=g)
    ids[1:4] = target[0:3].argmax(-1)
    cu = torch.arange(0, rows_max * n + 1, n, dtype=torch.int32, device=dev)
    r = mkv.verify_drafts(target.to(dev), ids.to(dev), cu, torch.tensor([0.0, 0.0, 0.0, 0.0] + [0.5] * 8, device=dev),
                          torch.empty(rows_max, V).exponential_(generator=g).to(dev), n, draft_logits=draft.to(dev))
    count = r.num_accepted.tolist()
    assert count[0] == n and all(1 <= x <= n for x in count)
    assert r.accepted.tolist() == [list(range(x)) + [-1] * (n - x) for x in count]
    pool.pages.compact(tables, t(before), r.accepted)
    lens.copy_(t(before) + r.num_accepted)
    pool.trim()
    for i in range(L):
        for b in range(rows_max):
            for xs in (lists[i][b].k, lists[i][b].v, lists[i][b].w):
                for h in range(H):
                    del xs[h][before[b] + count[b]:]
    compare()
    step([1, 1, 1])
    compare()


CFG = E.ModelConfig(vocab_size=512, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128,
                    intermediate_size=512, max_position=4096)


@pytest.mark.parametrize("use_graphs", [True, False])
@pytest.mark.parametrize("kv", ["auto", "fp8_per_tensor", "int8_per_token_head"])
def test_the_engine_accumulates(dev, use_graphs, kv):
    """Every row of a request gives one a query head: a KV head's weights sum to the
    group times the rows, in every layer; the tokens are those without weights."""
    announce(f"cache budget: the engine's weights, graphs {use_graphs}, {kv} KV")
    g = torch.Generator().manual_seed(41)
    prompts = [torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in (5, 70, 33)]

    def engine():
        model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
        model.fuse_decode_step = False
        return model, E.Engine(model, num_blocks=64, max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256,
                               kv_cache_dtype=kv, use_graphs=use_graphs)

    plain = engine()[1].generate(prompts, max_tokens=6)
    model, eng = engine()
    model.attach_attention_weights()
    reqs = [eng.add_request(p, 6) for p in prompts]
    blocks = {}
    while not eng.sched.done():
        eng.step()
        for r in reqs:
            if r.blocks:
                blocks[r.req_id] = list(r.blocks)
    assert [r.tokens[r.prompt_len:] for r in reqs] == plain
    for r in reqs:
        rows = len(r.tokens) - 1  # (the last token's K and V are not cached)
        n = torch.arange(rows)
        slots = (torch.tensor(blocks[r.req_id])[n // BS] * BS + n % BS).to(dev)
        for lay in model.layers:
            w = lay["attn"].attention_weights.flatten(0, 1)[slots].double().sum(0).cpu()
            want = CFG.num_heads // CFG.num_kv_heads * rows
            assert bool(((w - want).abs() <= 1e-4 * want).all()), (w, want)


def test_the_layer_s_routes(dev):
    """Full prefill, a chunk and a decode step through the layer, as the operator
    alone; a tree is refused, and so are steps without tables."""
    announce("cache budget: the attention layer's routes")
    g = torch.Generator().manual_seed(51)
    att = mkv.Attention(HQ, D, 1.0, H, BS)
    att.k_cache, att.v_cache = (torch.zeros(12, BS, H, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    att.attention_weights, att.weights_decay = torch.full((12, BS, H), 7.0, device=dev), 0.5
    want = att.attention_weights.clone()
    bt = torch.tensor([[3, 5, 1, -1], [0, 2, 4, 6]], dtype=torch.int32, device=dev)
    lens = [0, 0]
    for new, full in (([20, 33], True), ([9, 1], False), ([1, 1], None)):
        first, lens = lens, [a + b for a, b in zip(lens, new)]
        row = torch.tensor([r for r, n in enumerate(new) for _ in range(n)], device=dev)
        pos = torch.tensor([a + i for a, n in zip(first, new) for i in range(n)], device=dev)
        slots = bt[row, pos // BS].long() * BS + pos % BS
        q, k, v = (torch.randn(len(row), n, D, generator=g).to(dev, torch.bfloat16) for n in (HQ, H, H))
        cu = torch.tensor([0] + new, device=dev).cumsum(0).int()
        ctx = torch.tensor(lens, device=dev)
        C.set_context(full is not None, cu_seqlens_q=cu if full is not None else None, max_seqlen_q=max(new), slot_mapping=slots,
                      context_lens=ctx, block_tables=bt, positions=pos, is_full_prefill=bool(full))
        try:
            att(q, k, v)
        finally:
            C.reset_context()
        mkv.paged_attention_weights(q, att.k_cache, want, bt, ctx, D ** -0.5, HQ, H, D, BS,
                                    cu_seqlens_q=cu if full is not None else None, decay=0.5)
        assert torch.equal(att.attention_weights, want)
    C.set_context(True, cu_seqlens_q=cu, slot_mapping=slots, context_lens=ctx, block_tables=bt,
                  tree_mask=torch.ones(2, 1, dtype=torch.bool, device=dev))
    try:
        with pytest.raises(ValueError, match="not accumulated over trees"):
            att(q, k, v)
        C.set_context(True, cu_seqlens_q=cu, slot_mapping=slots, is_full_prefill=True)
        with pytest.raises(ValueError, match="require context_lens"):
            att(q, k, v)
    finally:
        C.reset_context()
