"""GPU tests of attention weights attached to the engine's model: when, and what is
refused before anything changes."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from mkv import context as C
from mkv import engine as E

pytestmark = pytest.mark.gpu

CFG = E.ModelConfig(vocab_size=512, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128,
                    intermediate_size=512, max_position=4096)
BS = 16


def engine(dev, model=None, use_graphs=True, kv="auto"):
    model = model or E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
    return model, E.Engine(model, num_blocks=64, max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256,
                           kv_cache_dtype=kv, use_graphs=use_graphs)


def given(model):
    return [float(lay["attn"].attention_weights.double().sum()) for lay in model.layers]


def test_not_behind_captured_steps(dev):
    """A captured step goes on as it was captured: weights attached behind it would
    miss every replay, and replays would write weights that were given up."""
    announce("weights attached: behind captured steps they are refused")
    prompt = torch.randint(0, CFG.vocab_size, (20,), generator=torch.Generator().manual_seed(1)).tolist()
    model, eng = engine(dev)
    eng.generate([prompt], max_tokens=4)
    with pytest.raises(RuntimeError, match="captured already"):
        model.attach_attention_weights()
    assert all(lay["attn"].attention_weights is None for lay in model.layers)
    # caches of a new engine: no step over them is captured
    _, eng = engine(dev, model)
    model.attach_attention_weights()
    model.attach_attention_weights(decay=0.5)
    eng.generate([prompt], max_tokens=4)
    kept = [lay["attn"].attention_weights for lay in model.layers]
    with pytest.raises(RuntimeError, match="captured already"):
        model.attach_attention_weights()
    assert all(lay["attn"].attention_weights is w for lay, w in zip(model.layers, kept))
    # steps that are not captured take them at any time: four rows of a request's
    # five decoded tokens follow
    model, eng = engine(dev, use_graphs=False)
    req = eng.add_request(prompt, 6)
    eng.step()
    eng.step()
    model.attach_attention_weights()
    while not eng.sched.done():
        eng.step()
    assert len(req.tokens) == 26
    for w in given(model):
        assert abs(w - 4 * CFG.num_heads) <= 1e-3


@pytest.mark.parametrize("kv", ["auto", "fp8_per_tensor", "int8_per_token_head"])
def test_a_refused_step_leaves_the_cache_as_it_was(dev, kv):
    """A tree, or a step without its lengths, over a model that accumulates: no K or V,
    no scale and no weight has changed."""
    announce(f"weights attached: refused steps change nothing, {kv} KV")
    model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
    model.attach_kv_cache(8, kv)
    model.attach_attention_weights()
    ids = torch.arange(6, device=dev)
    step = dict(cu_seqlens_q=torch.tensor([0, 6], dtype=torch.int32, device=dev), slot_mapping=ids, positions=ids,
                context_lens=torch.tensor([6], device=dev), max_seqlen_q=6,
                block_tables=torch.tensor([[0]], dtype=torch.int32, device=dev))

    def state():
        return [t.clone() for lay in model.layers for n in ("k_cache", "v_cache", "k_scale", "v_scale", "attention_weights")
                if (t := getattr(lay["attn"], n)) is not None]

    before = state()
    try:
        for change, what in ((dict(tree_mask=torch.ones(6, 6, dtype=torch.bool, device=dev)), "not accumulated over trees"),
                             (dict(context_lens=None), "require context_lens"), (dict(block_tables=None), "require context_lens")):
            C.set_context(True, **dict(step, **change))
            with pytest.raises(ValueError, match=what):
                model(ids, ids, ids)
            for a, b in zip(state(), before):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        C.set_context(True, **step)
        model(ids, ids, ids)
    finally:
        C.reset_context()
    for w in given(model):
        assert abs(w - 6 * CFG.num_heads) <= 1e-3


def test_an_engine_s_sequences_are_not_cut(dev):
    """It takes lengths and rotary positions from its host's token lists, which a cut
    would leave behind: its tables are refused, and nothing has changed."""
    announce("weights attached: the eviction refuses the engine's tables")
    prompt = torch.randint(0, CFG.vocab_size, (40,), generator=torch.Generator().manual_seed(2)).tolist()
    plain = engine(dev)[1].generate([prompt], max_tokens=6)
    model, eng = engine(dev)
    model.fuse_decode_step = False
    evict = model.attach_attention_weights()
    req = eng.add_request(prompt, 6)
    for _ in range(3):
        eng.step()
    before = [t.clone() for t in evict.tensors]
    for tables in (eng.meta.block_tables, eng.meta.block_tables[:2, :4]):
        with pytest.raises(ValueError, match="an Engine's sequences"):
            evict.evict(tables, eng.meta.seq_lens[:tables.shape[0]], 16)
    assert all(torch.equal(a, b) for a, b in zip(evict.tensors, before))
    while not eng.sched.done():
        eng.step()
    assert [req.tokens[40:]] == plain
    # the model without its engine: tables of the program's own
    model.attach_kv_cache(8, "auto")
    new = model.attach_attention_weights().evict(torch.tensor([[3, 1, 2]], dtype=torch.int32, device=dev),
                                                 torch.tensor([40], device=dev), 16)
    assert new.tolist() == [16]
