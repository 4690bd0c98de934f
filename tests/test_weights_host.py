"""What the attention weights' operator refuses, on the CPU: the wrapper's checks
and the library's own (which return before any launch)."""
from __future__ import annotations

import pytest
import torch

import mkv
from mkv import _lib
from mkv import context as C
from mkv import engine as E
from test_step_operators_host import lib, p  # noqa: F401  (lib: a fixture)


def weights(lib, **over):  # noqa: F811
    a = dict(w=p, decay=1.0, q=p, q_dt=_lib.DTYPE_BF16, k=p, kv_dt=_lib.DTYPE_BF16, blocks=8, ks=None, mode=0, bt=p,
             bt_stride=4, max_blocks=4, ctx=p, ctx_dt=1, cu=p, seqs=2, total=16, hq=8, hkv=4, d=128, bs=16, scale=0.1,
             ws=p, ws_bytes=1 << 20, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return lib.mkv_paged_weights(*a.values())


def test_refusals(lib):  # noqa: F811
    assert weights(lib, d=96) == -4 and weights(lib, hq=9) == -5 and weights(lib, hq=68) == -5
    assert weights(lib, bs=8) == -6 and weights(lib, bs=24) == -6
    assert weights(lib, q_dt=_lib.DTYPE_F16) == -3 and weights(lib, kv_dt=_lib.DTYPE_I8) == -3
    assert weights(lib, kv_dt=7) == -3 and weights(lib, mode=2) == -3 and weights(lib, ctx_dt=5) == -3
    assert weights(lib, kv_dt=_lib.DTYPE_FP8E4M3, q_dt=_lib.DTYPE_F32) == -3
    assert weights(lib, kv_dt=_lib.DTYPE_FP8E4M3) == -1
    for name in ("w", "q", "k", "bt", "ctx"):
        assert weights(lib, **{name: None}) == -1, name
    assert weights(lib, bt_stride=3) == -9 and weights(lib, q=p + 8) == -8 and weights(lib, k=p + 2) == -8
    assert weights(lib, w=p + 2) == -8 and weights(lib, ws=p + 8) == -8
    assert weights(lib, seqs=-1) == -2 and weights(lib, total=-1) == -2 and weights(lib, blocks=1 << 30) == -2
    assert weights(lib, max_blocks=1 << 28, bt_stride=1 << 28) == -2 and weights(lib, total=1 << 28) == -2
    assert weights(lib, hq=16384, hkv=1024) == -2
    # one row a sequence
    assert weights(lib, cu=None) == -2 and weights(lib, cu=None, total=2, seqs=2, w=None) == -1
    assert weights(lib, seqs=0) == 0 and weights(lib, max_blocks=0) == 0 and weights(lib, blocks=0) == 0
    need = lib.mkv_paged_weights_workspace_size(2, 16, 8, 4, 128, 16, 4, _lib.DTYPE_BF16, 0)
    assert need >= 16 * 8 * 4 and weights(lib, ws_bytes=need - 1) == -7
    assert lib.mkv_paged_weights_workspace_size(2, 2, 8, 4, 128, 16, 4, _lib.DTYPE_BF16, 1) == 0
    assert lib.mkv_paged_weights_workspace_size(2, 2, 8, 4, 128, 16, 4096, _lib.DTYPE_BF16, 1) > 0
    # (a grid past 2^32 threads)
    assert weights(lib, seqs=1 << 23, total=1 << 23, ws_bytes=1 << 62) == -2


def test_the_scores_room_is_bounded(lib):  # noqa: F811
    """Decode's kept scores follow the table's width: no more than 256 MiB of them,
    whatever the sequences and heads."""
    def room(seqs, hq, hkv, tokens):
        return lib.mkv_paged_weights_workspace_size(seqs, seqs, hq, hkv, 128, 16, tokens // 16, _lib.DTYPE_BF16, 1)

    # (of all pairs at once: 0.94 GiB, just over 1 GiB, 4 GiB)
    for seqs, hq, hkv, tokens in ((60, 16, 8, 131072), (64, 64, 8, 32768), (64, 64, 8, 131072), (1, 8, 1, 1 << 19)):
        assert 0 < room(seqs, hq, hkv, tokens) <= 256 << 20
    assert room(2, 32, 8, 131072) == 2 * 8 * 128 * 4 * (8 + 1024 * 4)
    # (one pair's would not fit: none are kept)
    assert 0 < room(1, 8, 1, 1 << 25) <= 1 << 22 and 0 < room(3, 4, 1, 1 << 25) <= 1 << 22


def test_work_past_whole_numbers_is_refused(lib):  # noqa: F811
    """The work of chunks is dealt out in doubles, which hold it exactly up to 2^53."""
    size = dict(seqs=1, hq=16, hkv=1, bs=1 << 20, blocks=8, ws_bytes=1 << 62)
    assert weights(lib, total=1 << 23, max_blocks=2047, bt_stride=2047, **size) == -2
    assert weights(lib, total=1 << 23, max_blocks=1, bt_stride=1, ws=None, **size) == -7


def test_the_wrapper_s_checks():
    q, k, w = torch.zeros(2, 8, 128), torch.zeros(4, 16, 8, 128), torch.zeros(4, 16, 8)
    bt, cl = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="no CPU fallback"):
        mkv.paged_attention_weights(q, k, w, bt, cl, 0.1, 8, 8, 128, 16)
    for decay in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="decay must be finite"):
            mkv.paged_attention_weights(q, k, w, bt, cl, 0.1, 8, 8, 128, 16, decay=decay)


def test_a_layer_refuses_a_step_ahead_of_its_store():
    """What cannot be accumulated is refused before the step's K and V go anywhere."""
    att = mkv.Attention(4, 64, 1.0, 2, 16)
    att.k_cache, att.v_cache = torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64)
    att.attention_weights = torch.zeros(4, 16, 2)
    q, k, v = torch.zeros(1, 4, 64), torch.zeros(1, 2, 64), torch.zeros(1, 2, 64)
    step = dict(slot_mapping=torch.zeros(1, dtype=torch.int64), context_lens=torch.ones(1, dtype=torch.int64),
                block_tables=torch.zeros(1, 1, dtype=torch.int32))
    chunk = dict(step, cu_seqlens_q=torch.tensor([0, 1], dtype=torch.int32))
    try:
        for prefill, c, decay, what in (
                (True, dict(chunk, tree_mask=torch.ones(1, 1, dtype=torch.bool)), 1.0, "not accumulated over trees"),
                (True, dict(chunk, context_lens=None), 1.0, "require context_lens"),
                (False, dict(step, block_tables=None), 1.0, "require context_lens"),
                (False, step, float("nan"), "must be finite")):
            att.weights_decay = decay
            C.set_context(prefill, **c)
            with pytest.raises(ValueError, match=what):
                att(q, k, v)
    finally:
        C.reset_context()


def test_the_model_refuses_weights_before_it_changes():
    cfg = E.ModelConfig(vocab_size=32, hidden_size=64, num_layers=1, num_heads=2, num_kv_heads=1, head_dim=64,
                        intermediate_size=64, max_position=64)
    model = E.Qwen3Model(cfg, "cpu", block_size=16)
    with pytest.raises(RuntimeError, match="attach_kv_cache comes first"):
        model.attach_attention_weights()
    model.attach_kv_cache(2, "auto")
    with pytest.raises(ValueError, match="must be finite"):
        model.attach_attention_weights(float("inf"))
    with pytest.raises(ValueError, match="no CPU fallback"):
        model.attach_attention_weights()
    assert model.layers[0]["attn"].attention_weights is None


@pytest.mark.parametrize("decay", [3.5e38, -1e300, float("-inf"), float("nan")])
def test_a_decay_that_float32_does_not_hold(decay):
    """It would reach the kernel as an infinity, and 0 times that is NaN."""
    q, k, w = torch.zeros(2, 8, 128), torch.zeros(4, 16, 8, 128), torch.zeros(4, 16, 8)
    bt, cl = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="decay must be finite"):
        mkv.paged_attention_weights(q, k, w, bt, cl, 0.1, 8, 8, 128, 16, decay=decay)
