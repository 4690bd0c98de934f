"""What the speculative step's operators refuse, on the CPU: the wrappers'
checks and the library's own (which return before any launch)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mkv
from mkv import _lib

p = 4096  # a pointer that is never read: every call below is refused before a launch


@pytest.fixture(scope="module")
def lib():
    try:
        return _lib.load()
    except RuntimeError:
        pytest.skip("libmkv.so not built")


def tree(lib, **over):
    a = dict(out=p, q=p, q_dt=_lib.DTYPE_BF16, k=p, v=p, kv_dt=_lib.DTYPE_BF16, blocks=8, ks=None, vs=None, mode=0, bt=p,
             bt_stride=4, max_blocks=4, ctx=p, ctx_dt=1, cu=p, mask=p, mask_stride=8, cols=8, seqs=2, total=16, hq=8, hkv=4,
             d=128, bs=16, scale=0.1, ws=p, ws_bytes=0, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return lib.mkv_paged_tree(*a.values())


def test_tree_refusals(lib):
    assert tree(lib, d=96) == -4 and tree(lib, d=64, hkv=1, hq=2) == -4
    assert tree(lib, hq=9) == -5 and tree(lib, hq=68) == -5 and tree(lib, d=64, hq=36) == -5
    assert tree(lib, bs=8) == -6 and tree(lib, bs=24) == -6
    assert tree(lib, q_dt=_lib.DTYPE_F16) == -3 and tree(lib, kv_dt=_lib.DTYPE_I8) == -3
    assert tree(lib, kv_dt=_lib.DTYPE_FP8E4M3, q_dt=_lib.DTYPE_F32) == -3
    assert tree(lib, kv_dt=_lib.DTYPE_FP8E4M3) == -1 and tree(lib, mode=2) == -3
    assert tree(lib, out=None) == -1 and tree(lib, mask=None) == -1 and tree(lib, bt=None) == -1
    assert tree(lib, bt_stride=3) == -9 and tree(lib, mask_stride=-1) == -9
    assert tree(lib, q=p + 8) == -8 and tree(lib, k=p + 2) == -8
    assert tree(lib, seqs=-1) == -2 and tree(lib, total=-1) == -2 and tree(lib, cols=-1) == -2
    assert tree(lib, max_blocks=1 << 28, bt_stride=1 << 28) == -2 and tree(lib, ctx_dt=7) == -3
    assert tree(lib, seqs=0) == 0 and tree(lib, total=0) == 0
    big = dict(max_blocks=4096, bt_stride=4096)
    need = lib.mkv_paged_tree_workspace_size(2, 16, 8, 4, 128, 16, 4096, 8, _lib.DTYPE_BF16)
    assert need > 0 and tree(lib, ws_bytes=need - 1, **big) == -7 and tree(lib, ws=None, **big) == -7


def test_logprobs_refusals(lib):
    def call(**over):
        a = dict(lp=p, ent=p, top_lp=p, top_ids=p, logits=p, stride=100, dt=_lib.DTYPE_BF16, rows=3, vocab=100, ids=p,
                 ids_stride=2, n=2, ids_dt=1, top=5, ws=p, ws_bytes=1 << 20, stream=None)
        assert set(over) <= set(a)
        a.update(over)
        return lib.mkv_token_logprobs(*a.values())

    assert call(top=65) == -2 and call(vocab=4, top=5) == -2 and call(vocab=0) == -2 and call(rows=-1) == -2
    assert call(stride=99) == -9 and call(ids_stride=1) == -9
    assert call(ids=None) == -1 and call(ent=None) == -1 and call(top_ids=None) == -1 and call(ws=None) == -1
    assert call(dt=_lib.DTYPE_I8) == -3 and call(ids_dt=5) == -3
    assert call(logits=p + 1) == -8 and call(ws=p + 4) == -8 and call(ws_bytes=16) == -7
    assert call(rows=0) == 0


def test_pages_refusals(lib):
    ptrs, rows = (ctypes.c_void_p * 2)(p, p + 4096), (ctypes.c_int64 * 2)(32, 32)
    bad_rows, bad_ptrs = (ctypes.c_int64 * 2)(32, 6), (ctypes.c_void_p * 2)(p, None)
    odd = (ctypes.c_void_p * 2)(p, p + 2)
    ok = [ctypes.addressof(ptrs), ctypes.addressof(rows), 2, 10, 16]

    def pools(ptrs=ptrs, rows=rows, n=2, pages=10, bs=16):
        return [ctypes.addressof(ptrs), ctypes.addressof(rows), n, pages, bs]

    def copy(pool=ok, src=p, dst=p, dt=1, n=3):
        return lib.mkv_copy_pages(*pool, src, dst, dt, n, None)

    assert copy(pools(rows=bad_rows)) == -2 and copy(pools(ptrs=bad_ptrs)) == -1 and copy(pools(ptrs=odd)) == -8
    assert copy(pools(bs=0)) == -2 and copy(pools(pages=1 << 31)) == -2 and copy([None] + ok[1:]) == -1
    assert copy(src=None) == -1 and copy(dt=3) == -3 and copy(n=-1) == -2 and copy(n=0) == 0

    def compact(pool=ok, bt=p, stride=4, blocks=4, pre=p, pre_dt=1, acc=p, acc_dt=1, acc_stride=5, batch=2, n=5):
        return lib.mkv_compact_slots(*pool, bt, stride, blocks, pre, pre_dt, acc, acc_dt, acc_stride, batch, n, None)

    assert compact(pools(bs=12)) == -6 and compact(n=2049, acc_stride=4000) == -2 and compact(batch=70000) == -2
    assert compact(stride=3) == -9 and compact(acc_stride=4) == -9 and compact(bt=None) == -1 and compact(acc_dt=2) == -3
    assert compact(batch=0) == 0 and compact(n=0, acc_stride=0) == 0

    def assign(pool=ok, bt=p, stride=4, blocks=4, lens=p, held=p, refs=p, par=p, par_dt=1, tok=p, tok_dt=1, ok_=p, rows=6,
               ws=p, n=1 << 20):
        return lib.mkv_assign_pages(*pool, bt, stride, blocks, lens, held, refs, par, par_dt, tok, tok_dt, ok_, rows, ws, n,
                                    None)

    need = lib.mkv_assign_pages_workspace_size(6, 4)
    assert assign(rows=1025) == -2 and assign(pools(bs=12)) == -6 and assign(stride=3) == -9 and assign(n=need - 1) == -7
    assert assign(par=None) == -1 and assign(held=None) == -1 and assign(par_dt=2) == -3 and assign(tok_dt=2) == -3
    assert assign(blocks=1 << 30, stride=1 << 30) == -2 and assign(rows=0) == 0


def test_wrappers_refuse_cpu_tensors():
    q, kc = torch.zeros(2, 8, 128), torch.zeros(1, 16, 8, 128)
    bt, cl, cu = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int64), torch.tensor([0, 2])
    with pytest.raises(ValueError, match="no CPU fallback"):
        mkv.paged_attention_tree(q, kc, kc, bt, cl, cu, torch.ones(2, 2, dtype=torch.bool), 0.1, 8, 8, 128, 16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        mkv.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="no CPU fallback"):
        mkv.CachePages([kc])
    with pytest.raises(ValueError, match="no cache tensors"):
        mkv.CachePages([])


def test_context_carries_the_tree_mask():
    from mkv import context as C

    m = torch.ones(2, 2, dtype=torch.bool)
    C.set_context(True, tree_mask=m)
    assert C.get_context().tree_mask is m
    C.reset_context()
    assert C.get_context().tree_mask is None
