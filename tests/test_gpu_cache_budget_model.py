"""GPU tests of a model within a cache budget, as a program of its own drives it.

* Greedy generation by captured decode steps, sequences cut between them and their pages
  given back, the rotary positions going on from the uncut lengths: against the model in
  float64 on the CPU over lists of keys, values and weights per layer and head.
* Forked and compacted rows take their weights along where the page operators have them.
* Weights of verified drafts: the accepted rows' alone.

Logits: a float32 product of up to 512 terms is off by 512 * 2^-24 = 3e-5 of its terms'
sizes, and some ten of them follow each other, so that the normalised hidden state, of
size 1, is off by 3e-4 at most; a logit sums 256 of its terms times weights of 0.02: 1.2e-3
at most.
"""
from __future__ import annotations

import math

import pytest
import torch

import mkv
from conftest import announce
from mkv import context as C
from mkv import engine as E
from mkv.decode_state import DecodeGraphs, DecodeMetadata
from test_gpu_cache_budget import BS, CFG, D, G, H, HQ, Lists

pytestmark = pytest.mark.gpu


class Model64:
    """The decoder in float64, one sequence a call, over lists of its tokens."""

    def __init__(self, model):
        self.m = model
        self.w = {n: t.cpu().double() for n, t in (("embed", model.embed), ("final", model.final_norm), ("cs", model.cos_sin))}
        self.layers = [{n: t.cpu().double() for n, t in lay.items() if n != "attn"} for lay in model.layers]

    def norm(self, x, weight):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.m.cfg.eps) * weight

    def rotate(self, x, pos):
        cos, sin = self.w["cs"][pos][:, None].chunk(2, -1)
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def logits(self, lists, tokens, pos, decay):
        n, pos = len(tokens), torch.tensor(pos)
        x = self.w["embed"][torch.tensor(tokens)]
        for one, lay in zip(lists, self.layers):
            q, k, v = (self.norm(x, lay["in_norm"]) @ lay["qkv"].t()).split([HQ * D, H * D, H * D], -1)
            q = self.rotate(self.norm(q.reshape(n, HQ, D), lay["q_norm"]), pos)
            k = self.rotate(self.norm(k.reshape(n, H, D), lay["k_norm"]), pos)
            for i in range(n):
                one.append(k[i], v.reshape(n, H, D)[i])
            x = x + one.attend(q, n, decay).reshape(n, HQ * D) @ lay["o"].t()
            gate, up = (self.norm(x, lay["post_norm"]) @ lay["gate_up"].t()).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ lay["down"].t()
        return self.norm(x, self.w["final"]) @ self.w["embed"].t()


def test_generation_goes_on_across_cuts(dev):
    announce("cache budget: captured generation across cuts, fp32")
    pages, max_rows, width, budget, sinks, recent, decay = 24, 3, 8, 40, 2, 8, 0.95
    model = E.Qwen3Model(CFG, dev, dtype=torch.float32, seed=5, block_size=BS)
    model.attach_kv_cache(pages, "auto")
    evict = model.attach_attention_weights(decay)
    meta = DecodeMetadata(max_rows, width, BS, pages, dev)
    pool = mkv.PagePool(meta.block_tables, meta.seq_lens, mkv.CachePages(evict.tensors))
    oracle = Model64(model)
    g = torch.Generator().manual_seed(61)
    seqs = [torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in (50, 23)]
    lists = [[Lists() for _ in model.layers] for _ in seqs]
    rows = len(seqs)

    def t(x, dtype=torch.int64):
        return torch.tensor(x, dtype=dtype, device=dev)

    def same(logits):
        """Against the model in float64, on what each row has had since."""
        for r in range(rows):
            new = seqs[r][done[r]:]
            want = oracle.logits(lists[r], new, range(done[r], len(seqs[r])), decay)[-1]
            assert float((logits[r].cpu().double() - want).abs().max()) <= 1.2e-3
            done[r] = len(seqs[r])

    done = [0] * rows
    stay = t([0, 1, -1])
    lens = [len(s) for s in seqs]
    assert pool.assign(stay, t(lens + [0])).tolist() == [True] * max_rows
    row = t([r for r, n in enumerate(lens) for _ in range(n)])
    pos = t([i for n in lens for i in range(n)])
    slots = meta.block_tables[row, pos // BS].long() * BS + pos % BS
    cu = t([0] + lens, torch.int32).cumsum(0).int()
    C.set_context(True, cu_seqlens_q=cu, max_seqlen_q=max(lens), slot_mapping=slots, context_lens=t(lens),
                  block_tables=meta.block_tables[:rows], positions=pos)
    try:
        hidden = model(t([x for s in seqs for x in s]), pos, slots)
    finally:
        C.reset_context()
    logits = model.logits(hidden[cu[1:].long() - 1])
    meta.seq_lens[:rows] = t(lens)
    same(logits)

    # decode steps: the positions are the program's own, and no cut sets them back
    ids, out = torch.zeros(max_rows, dtype=torch.int64, device=dev), torch.zeros(max_rows, CFG.vocab_size, device=dev)
    positions = meta.seq_lens.clone()

    def step_fn(rows, slot, ctx, bt):
        C.set_context(False, slot_mapping=slot, context_lens=ctx, block_tables=bt)
        try:
            out[:rows].copy_(model.logits(model(ids[:rows], positions[:rows], slot)))
            positions[:rows] += ctx > 0
        finally:
            C.reset_context()

    graphs = DecodeGraphs(meta, step_fn, buckets=[max_rows])
    graphs.capture()
    assert positions.tolist() == lens + [0]
    cuts = 0
    for turn in range(30):
        tok = logits.argmax(-1)
        for r, x in enumerate(tok.tolist()):
            seqs[r].append(x)
        ids[:rows] = tok
        assert pool.assign(stay, meta.seq_lens + 1).tolist() == [True] * max_rows
        graphs.run(rows)
        logits = out[:rows].clone()
        same(logits)
        if turn % 9 != 4:
            continue
        # kept tokens by the device's own weights, which are close to the lists'
        n = meta.seq_lens.tolist()
        for i, lay in enumerate(model.layers):
            w = lay["attn"].attention_weights.flatten(0, 1)
            for r in range(rows):
                at = torch.arange(n[r], device=dev)
                have = w[meta.block_tables[r, at // BS].long() * BS + at % BS].cpu()
                for h in range(H):
                    assert len(lists[r][i].w[h]) == n[r]
                    want = torch.tensor(lists[r][i].w[h], dtype=torch.float64)
                    assert float((have[:, h].double() - want).abs().max()) <= 1e-3 * max(1.0, float(want.max()))
                    lists[r][i].w[h] = have[:, h].tolist()
                if n[r] > budget:
                    lists[r][i].keep(lists[r][i].choose(budget, sinks, recent)[0])
        cuts += sum(x > budget for x in n)
        meta.seq_lens.copy_(evict.evict(meta.block_tables, meta.seq_lens, budget, sinks=sinks, recent=recent))
        pool.trim()
        assert pool.held.tolist() == [-(-min(x, budget) // BS) for x in n]
    assert cuts >= 4 and positions.tolist() == [len(s) for s in seqs] + [0]


def test_weights_go_with_forked_and_compacted_rows(dev):
    """A part-filled page that a fork copies, and accepted rows that move up, bring
    their weights (and scales) where the page operators were given them."""
    announce("cache budget: forks and compactions with weights")
    g = torch.Generator().manual_seed(62)
    model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
    model.attach_kv_cache(16, "int8_per_token_head")
    evict = model.attach_attention_weights()
    for x in evict.tensors:
        x.copy_(torch.rand(x.shape, generator=g) * 50)
    tables, lens = torch.zeros(3, 5, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    pool = mkv.PagePool(tables, lens, mkv.CachePages(evict.tensors))

    def t(*x):
        return torch.tensor(x, dtype=torch.int64, device=dev)

    def rows(r, n):
        at = torch.arange(n, device=dev)
        slots = tables[r, at // BS].long() * BS + at % BS
        return [x.flatten(0, 1)[slots].clone() for x in evict.tensors]

    assert len(evict.tensors) == 5 * CFG.num_layers
    assert pool.assign(t(0, -1, -1), t(45, 0, 0)).tolist() == [True] * 3
    lens.copy_(t(37, 0, 0))
    before = rows(0, 45)
    assert pool.fork(0, [1]).tolist() == [True] * 3
    assert pool.assign(t(0, 1, -1), t(45, 45, 0)).tolist() == [True] * 3
    assert tables[0, 2] != tables[1, 2]
    for got, want in zip(rows(1, 37), before):
        assert torch.equal(got, want[:37])
    pool.pages.compact(tables, t(37, 37, 0), t(0, 3, 6, -1, 1, 2, -1, -1, -1, -1, -1, -1).reshape(3, 4))
    for got, want in zip(rows(0, 40), before):
        assert torch.equal(got, want[list(range(37)) + [37, 40, 43]])


@pytest.mark.parametrize("accepted", [[0, 1, 2], [0], [0, 2, 5], [0, 1, 2, 3, 4, 5]])
def test_weights_of_accepted_drafts_alone(dev, accepted):
    """Weights accumulated once the drafts are verified and compacted, by the accepted
    rows: as if no other had been there."""
    announce(f"cache budget: weights of accepted drafts {accepted}")
    g = torch.Generator().manual_seed(63)
    prefix, drafted, n = 30, 6, len(accepted)
    k_cache, v_cache, weights = (torch.zeros(*s, device=dev) for s in ((6, BS, H, D), (6, BS, H, D), (6, BS, H)))
    table = torch.tensor([[4, 1, 5]], dtype=torch.int32, device=dev)
    pages, at = mkv.CachePages([k_cache, v_cache, weights]), torch.arange(prefix + drafted, device=dev)
    slots = table[0, at // BS].long() * BS + at % BS
    q, k, v = (torch.randn(prefix + drafted, x, D, generator=g) for x in (HQ, H, H))
    lists = Lists()

    def accumulate(rows, length):
        mkv.paged_attention_weights(q[rows].to(dev), k_cache, weights, table, torch.tensor([length], device=dev), 1 / math.sqrt(D),
                                    HQ, H, D, BS, cu_seqlens_q=torch.tensor([0, len(rows)], dtype=torch.int32, device=dev),
                                    decay=0.9)

    mkv.store_kvcache(k.to(dev), v.to(dev), k_cache, v_cache, slots, BS)
    accumulate(list(range(prefix)), prefix)
    for i in range(prefix):
        lists.append(k[i], v[i])
    lists.attend(q[:prefix], prefix, 0.9)
    pages.compact(table, torch.tensor([prefix], device=dev), torch.tensor([accepted], device=dev))
    rows = [prefix + i for i in accepted]
    accumulate(rows, prefix + n)
    for i in rows:
        lists.append(k[i], v[i])
    lists.attend(q[rows], n, 0.9)
    for h in range(H):
        got = weights.flatten(0, 1)[slots[:prefix + n], h].cpu().double()
        want = torch.tensor(lists.w[h], dtype=torch.float64)
        # (a score is off by D 2^-24 of its terms' sizes, below 1e-4, twice in a weight)
        assert float(((got - want).abs() / want).max()) <= 3e-4
