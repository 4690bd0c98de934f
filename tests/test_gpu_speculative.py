"""GPU tests of the speculative step's operators together, as a program uses
them, and of the engine's log probabilities.

* A prompt's pages are forked, trees of drafted tokens are appended and
  verified by one forward over their masks, the accepted tokens' cache rows
  are moved up, tables fork again and rows are freed: the tokens are those of
  greedy decoding by whole prefills in another model, and so are the logits.
* The engine reports the log probabilities of the tokens it samples.
"""
from __future__ import annotations

import pytest
import torch

import mkv
from conftest import announce
from mkv import context as C
from mkv import engine as E
from mkv.decode_state import DecodeMetadata

pytestmark = pytest.mark.gpu

CFG = E.ModelConfig(vocab_size=512, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=2,
                    head_dim=128, intermediate_size=512, max_position=4096)
BS = 16


class Greedy:
    """Greedy continuation by whole prefills (fresh K and V, no pages read)."""

    def __init__(self, dev):
        self.dev = dev
        self.model = E.Qwen3Model(CFG, dev, dtype=torch.float32, seed=5, block_size=BS)
        self.model.attach_kv_cache(16, "auto")
        self.known = {}

    def logits(self, tokens):
        n, d = len(tokens), self.dev
        pos = torch.arange(n, device=d)
        cu = torch.tensor([0, n], dtype=torch.int32, device=d)
        C.set_context(True, cu_seqlens_q=cu, max_seqlen_q=n, slot_mapping=pos,
                      context_lens=torch.tensor([n], device=d),
                      block_tables=torch.arange(16, dtype=torch.int32, device=d)[None], positions=pos,
                      is_full_prefill=True)
        try:
            hidden = self.model(torch.tensor(tokens, device=d), pos, pos, full_prefill=True)
        finally:
            C.reset_context()
        return self.model.logits(hidden)[-1]

    def next(self, tokens):
        key = tuple(tokens)
        if key not in self.known:
            self.known[key] = int(self.logits(tokens).argmax())
        return self.known[key]


class Tree:
    """A drafted tree: node 0 is the sequence's last token, whose K and V are
    not cached yet; parent[i] < i."""

    def __init__(self, tokens, parent):
        self.tokens, self.parent = tokens, parent
        self.path = [[0]]
        for i, p in enumerate(parent[1:], 1):
            self.path.append(self.path[p] + [i])

    def mask_row(self, i, width):
        return [j in self.path[i] for j in range(width)]

    def depth(self, i):
        return len(self.path[i]) - 1


def _draft(greedy, seq, right, extra):
    """`right` tokens of the greedy continuation behind the last one, a wrong
    sibling beside each, and `extra` wrong tokens behind the last."""
    tokens, parent, at, line = [seq[-1]], [-1], 0, list(seq)
    for _ in range(right):
        good = greedy.next(line)
        tokens += [(good + 7) % CFG.vocab_size, good]
        parent += [at, at]
        at = len(tokens) - 1
        line.append(good)
    for _ in range(extra):
        tokens.append((greedy.next(line) + 11) % CFG.vocab_size)
        parent.append(at)
    return Tree(tokens, parent)


def test_forked_sequences_decode_speculatively_as_greedily(dev):
    announce("speculative: fork, tree attention, log probabilities, compaction against greedy decoding, fp32")
    greedy = Greedy(dev)
    model = E.Qwen3Model(CFG, dev, dtype=torch.float32, seed=5, block_size=BS)
    model.attach_kv_cache(48, "auto")
    meta = DecodeMetadata(4, 12, BS, 48, dev)
    caches = [t for lay in model.layers for t in (lay["attn"].k_cache, lay["attn"].v_cache)]
    pool = mkv.PagePool(meta.block_tables, meta.seq_lens, mkv.CachePages(caches))

    def t(x, dtype=torch.int64):
        return torch.tensor(x, dtype=dtype, device=dev)

    def forward(trees, lens):
        """One forward of every row's tree behind its lens[r] cached tokens."""
        width = max(len(x.tokens) for x in trees)
        ids = t([tok for x in trees for tok in x.tokens])
        pos = t([n + x.depth(i) for x, n in zip(trees, lens) for i in range(len(x.tokens))])
        # each drafted token's cache row: behind the prefix, in the tree's order
        at = t([n + i for x, n in zip(trees, lens) for i in range(len(x.tokens))])
        row = t([r for r, x in enumerate(trees) for _ in x.tokens])
        slots = meta.block_tables[row, at // BS].long() * BS + at % BS
        cu = [0]
        for x in trees:
            cu.append(cu[-1] + len(x.tokens))
        mask = t([x.mask_row(i, width) for x in trees for i in range(len(x.tokens))], torch.bool)
        C.set_context(True, cu_seqlens_q=t(cu, torch.int32), max_seqlen_q=width, slot_mapping=slots,
                      context_lens=t([n + len(x.tokens) for x, n in zip(trees, lens)]),
                      block_tables=meta.block_tables[:len(trees)], positions=pos, tree_mask=mask)
        try:
            hidden = model(ids, pos, slots)
        finally:
            C.reset_context()
        return model.logits(hidden), cu

    # the prompt, in row 0 (a chain is a tree)
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, CFG.vocab_size, (37,), generator=g).tolist()
    assert pool.assign(t([0, -1, -1, -1]), t([37, 0, 0, 0])).tolist() == [True] * 4
    logits, _ = forward([Tree(prompt, [i - 1 for i in range(37)])], [0])
    meta.seq_lens[0] = 37
    want = greedy.logits(prompt)
    assert float((logits[-1] - want).abs().max()) <= 3e-2
    first = mkv.token_logprobs(logits[-1:], logits[-1:].argmax(-1), top=3).top_indices[0].tolist()
    assert first == want.topk(3).indices.tolist()

    # three continuations of it, and one more row later
    assert pool.fork(0, [1, 2]).tolist() == [True] * 4
    tables = meta.block_tables.tolist()
    assert tables[0][:2] == tables[1][:2] == tables[2][:2] and len({x[2] for x in tables[:3]}) == 3
    seqs = [prompt + [tok] for tok in first]
    plan = [[(2, 1), (0, 2), (3, 0)], [(1, 1), (4, 2), (0, 0)], [(2, 0), (1, 3), (3, 1), (0, 4)], [(0, 1), (5, 0), (2, 2), (1, 0)]]
    accepted_in_all = 0
    for step, shapes in enumerate(plan):
        if step == 2:  # row 3 goes on with row 1's sequence, and row 2 with row 0's
            assert pool.assign(t([0, 1, 0, 1])).tolist() == [True] * 4
            seqs = [list(seqs[0]), list(seqs[1]), list(seqs[0]), list(seqs[1])]
        rows = len(seqs)
        lens = [len(s) - 1 for s in seqs]
        assert meta.seq_lens[:rows].tolist() == lens
        trees = [_draft(greedy, s, *shape) for s, shape in zip(seqs, shapes)]
        grow = [n + len(x.tokens) for n, x in zip(lens, trees)] + [0] * (4 - rows)
        parents = list(range(rows)) + [-1] * (4 - rows)
        assert pool.assign(t(parents), t(grow)).tolist() == [True] * 4
        logits, cu = forward(trees, lens)
        best = mkv.token_logprobs(logits, torch.full((cu[-1],), -1, device=dev), top=1).top_indices[:, 0].tolist()
        paths = []
        for r, x in enumerate(trees):
            at = 0
            path = [0]
            while True:
                good = best[cu[r] + at]
                kids = [i for i, p in enumerate(x.parent) if p == at and x.tokens[i] == good]
                if not kids:
                    break
                at = kids[0]
                path.append(at)
            paths.append(path)
            assert len(path) == 1 + shapes[r][0], f"step {step}, row {r}: {path}"
            # the path's tokens and one more of the model's own
            seqs[r] += [x.tokens[i] for i in path[1:]] + [best[cu[r] + at]]
            assert seqs[r][-1] == greedy.next(seqs[r][:-1])
        # log probabilities of every drafted token given its parent
        child = t([cu[r] + p for r, x in enumerate(trees) for p in x.parent[1:]])
        toks = t([tok for x in trees for tok in x.tokens[1:]])
        got = mkv.token_logprobs(logits[child], toks).logprobs.double()
        want = torch.log_softmax(logits[child].double(), -1).gather(1, toks[:, None])[:, 0]
        assert float((got - want).abs().max()) <= 1e-5
        # accepted rows move up behind the prefix
        most = max(len(p) for p in paths)
        accepted_in_all += sum(len(p) for p in paths)
        pool.pages.compact(meta.block_tables, t(lens), t([p + [-1] * (most - len(p)) for p in paths]))
        meta.seq_lens[:rows] = t([n + len(p) for n, p in zip(lens, paths)])
    assert accepted_in_all == sum(1 + right for shapes in plan for right, _ in shapes)

    # a plain decode step behind it all, over pages handed to the next token
    lens = [len(s) - 1 for s in seqs]
    assert pool.assign(t([0, 1, 2, 3]), t([n + 1 for n in lens])).tolist() == [True] * 4
    slot, ctx, bt = meta.step(4)
    C.set_context(False, slot_mapping=slot, context_lens=ctx, block_tables=bt)
    try:
        hidden = model(t([s[-1] for s in seqs]), ctx - 1, slot)
    finally:
        C.reset_context()
    logits = model.logits(hidden)
    for r, s in enumerate(seqs):
        want = greedy.logits(s)
        assert int(want.argmax()) == int(logits[r].argmax())
        assert float((logits[r] - want).abs().max()) <= 3e-2
    pages = pool.ref_counts.tolist()
    held = pool.held.tolist()
    assert sum(pages) == sum(held)
    for r in range(4):
        for page in meta.block_tables[r, :held[r]].tolist():
            assert pages[page] > 0
    pool.free(range(4))
    assert not any(pool.ref_counts.tolist()) and not any(meta.seq_lens.tolist())


@pytest.mark.parametrize("use_graphs", [True, False])
def test_engine_reports_log_probabilities(dev, use_graphs):
    announce(f"engine: log probabilities of the sampled tokens, graphs {use_graphs}")
    g = torch.Generator().manual_seed(21)
    prompts = [torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in (5, 70, 33, 18, 90)]
    wants = [None, 0, 3, 64, None]

    def engine():
        model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
        return E.Engine(model, num_blocks=96, max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256,
                        use_graphs=use_graphs)

    plain = engine().generate(prompts, max_tokens=6)
    eng = engine()
    with pytest.raises(ValueError, match="logprobs 65"):
        eng.add_request(prompts[0], 6, logprobs=65)
    with pytest.raises(ValueError, match="logprobs -1"):
        eng.add_request(prompts[0], 6, logprobs=-1)
    reqs = [eng.add_request(p, 6, logprobs=n) for p, n in zip(prompts, wants)]
    while not eng.sched.done():
        before = [(r, len(r.reports)) for r in reqs]
        eng.step()
        if not eng.last_sampled:
            continue
        x = torch.log_softmax(eng.last_logits.double(), -1)
        entropy = -(x.exp() * x).sum(-1)
        new = [(r, r.reports[n]) for r, n in before if len(r.reports) > n]
        for r, rep in new:
            tok = r.tokens[-1]
            near = ((x[:, tok] - rep.logprob).abs() <= 1e-5) & ((entropy - rep.entropy).abs() <= 1e-4)
            rows = [i for i in near.nonzero()[:, 0].tolist() if eng.last_sampled[i] == tok]
            assert rows, f"request {r.req_id}: no row of the step has {rep.logprob}, {rep.entropy}"
            i = rows[0]
            assert len(rep.top) == r.logprobs
            order = torch.sort(eng.last_logits[i].float(), descending=True, stable=True).indices[:r.logprobs].tolist()
            assert [j for j, _ in rep.top] == order
            assert all(abs(float(x[i, j]) - lp) <= 1e-5 for j, lp in rep.top)
    assert [r.tokens[r.prompt_len:] for r in reqs] == plain, "reports change no token"
    assert [len(r.reports) for r in reqs] == [0 if n is None else 6 for n in wants]


def test_engine_reports_survive_a_preemption(dev):
    """A pool too small for all sequences: preempted requests start again from
    their tokens, and keep one report a generated token."""
    announce("engine: log probabilities with preemptions")
    g = torch.Generator().manual_seed(22)
    prompts = [torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in (40, 44, 47, 30)]
    model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
    eng = E.Engine(model, num_blocks=14, max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256)
    reqs = [eng.add_request(p, 24, logprobs=2) for p in prompts]
    while not eng.sched.done():
        eng.step()
    assert eng.sched.num_preemptions > 0
    for r in reqs:
        assert r.num_generated == len(r.reports) == 24
        for tok, rep in zip(r.tokens[r.prompt_len:], r.reports):
            assert rep.logprob <= rep.top[0][1] and rep.top[0][1] >= rep.top[1][1] and rep.entropy >= -1e-4
            assert tok != rep.top[0][0] or abs(rep.logprob - rep.top[0][1]) <= 1e-5


@pytest.mark.parametrize("kv", ["auto", "fp8_per_tensor", "fp8_per_token_head", "int8_per_token_head"])
def test_a_chain_gives_the_chunked_prefill_s_logits(dev, kv):
    """Two sequences' next tokens over each cache format, once as a chunk of a
    prompt and once as a tree that is a chain: the same K and V are appended to the
    same rows, and the logits agree to the roundings of bf16 activations (the bound
    that the engine's logits meet against another attention)."""
    announce(f"speculative: a chain against a prefill chunk, {kv} KV")
    model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
    model.attach_kv_cache(12, kv)
    g = torch.Generator().manual_seed(9)
    lens, new = [40, 21], [9, 4]
    tables = torch.tensor([[3, 7, 1, 5], [2, 9, 4, 0]], dtype=torch.int32)
    toks = [torch.randint(0, CFG.vocab_size, (n + m,), generator=g) for n, m in zip(lens, new)]

    def step(first, last, tree):
        ids = torch.cat([x[a:b] for x, a, b in zip(toks, first, last)])
        pos = torch.cat([torch.arange(a, b) for a, b in zip(first, last)])
        row = torch.cat([torch.full((b - a,), r) for r, (a, b) in enumerate(zip(first, last))])
        slots = (tables[row, pos // BS].long() * BS + pos % BS).to(dev)
        sizes = [b - a for a, b in zip(first, last)]
        cu = torch.tensor([0, sizes[0], sum(sizes)], dtype=torch.int32, device=dev)
        mask = None
        if tree:
            mask = torch.ones(sum(sizes), max(sizes), dtype=torch.bool)
            local = torch.cat([torch.arange(n) for n in sizes])
            mask &= torch.arange(max(sizes))[None] <= local[:, None]
            mask = mask.to(dev)
        C.set_context(True, cu_seqlens_q=cu, max_seqlen_q=max(sizes), slot_mapping=slots,
                      context_lens=torch.tensor(last, device=dev), block_tables=tables.to(dev), positions=pos.to(dev),
                      tree_mask=mask)
        try:
            return model.logits(model(ids.to(dev), pos.to(dev), slots)).float()
        finally:
            C.reset_context()

    step([0, 0], lens, False)
    ends = [n + m for n, m in zip(lens, new)]
    want = step(lens, ends, False)
    got = step(lens, ends, True)
    tol = 6e-2 + torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -14))) - 7)
    diff = (got - want).abs()
    print(f"max difference {float(diff.max()):.2e}, mean {float(diff.mean()):.2e}")
    assert bool((diff <= tol).all()) and float(diff.mean()) <= 1e-2
