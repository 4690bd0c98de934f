"""What the eviction and the page table's trim refuse, on the CPU: the wrappers'
checks and the library's own (which return before any launch)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mkv
from mkv import _lib
from test_step_operators_host import lib, p  # noqa: F401  (lib: a fixture)


def evict(lib, **over):  # noqa: F811
    n = 3
    ptrs, layers = (ctypes.c_void_p * n)(p, p, p), (ctypes.c_int * n)(0, 0, 0)
    a = dict(tensors=ctypes.addressof(ptrs), bytes=(ctypes.c_int64 * n)(256, 256, 4), layers=ctypes.addressof(layers), n=n,
             weights=ctypes.addressof(ptrs), num_layers=1, pages=10, bs=16, heads=2, bt=p, stride=4, blocks=4, lens=p,
             lens_dt=1, batch=2, budget=8, sinks=1, recent=2, new=p, ws=p, ws_bytes=1 << 20, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    if not isinstance(a["bytes"], (int, type(None))):
        keep = a["bytes"]
        a["bytes"] = ctypes.addressof(keep)
    return lib.mkv_evict_tokens(*a.values())


def test_evict_refusals(lib):  # noqa: F811
    assert evict(lib, bs=24) == -6 and evict(lib, bs=2) == -6 and evict(lib, heads=0) == -2 and evict(lib, heads=1025) == -2
    assert evict(lib, batch=70000) == -2 and evict(lib, budget=0) == -2 and evict(lib, sinks=-1) == -2
    assert evict(lib, sinks=5, recent=4) == -2 and evict(lib, recent=2 ** 31 - 1) == -2
    assert evict(lib, pages=1 << 28) == -2 and evict(lib, blocks=1 << 28, stride=1 << 28) == -2
    for name in ("tensors", "bytes", "layers", "weights", "bt", "lens", "new", "ws"):
        assert evict(lib, **{name: None}) == -1, name
    assert evict(lib, stride=3) == -9 and evict(lib, lens_dt=4) == -3 and evict(lib, ws=p + 2) == -8
    for size in (0, 6, 2052):
        assert evict(lib, bytes=(ctypes.c_int64 * 3)(256, size, 4)) == -2
    assert evict(lib, layers=ctypes.addressof((ctypes.c_int * 3)(0, 0, 1))) == -2
    assert evict(lib, tensors=ctypes.addressof((ctypes.c_void_p * 3)(p, p + 2, p))) == -8
    assert evict(lib, weights=ctypes.addressof((ctypes.c_void_p * 1)(None))) == -1
    need = lib.mkv_evict_tokens_workspace_size(1, 2, 2, 16, 4, 8)
    assert need == 2 * 2 * 8 * 4 and evict(lib, ws_bytes=need - 1) == -7
    assert lib.mkv_evict_tokens_workspace_size(1, 2, 2, 16, 1024, 8) == 2 * 2 * (8 + 16384) * 4
    assert evict(lib, batch=0) == 0 and evict(lib, num_layers=0, n=0) == 0
    # (a grid past 2^32 threads)
    assert evict(lib, batch=65535, heads=1024, ws_bytes=1 << 62) == -2


def test_the_keys_room_is_bounded(lib):  # noqa: F811
    """What long tables take follows their width: no more than 256 MiB beside the kept
    tokens' slots, whatever the layers and sequences, or what one sequence of a layer
    takes."""
    def keys(layers, batch, heads, blocks, budget=256):
        return lib.mkv_evict_tokens_workspace_size(layers, batch, heads, 16, blocks, budget) - layers * batch * heads * budget * 4

    assert keys(28, 60, 8, 131072 // 16) <= 256 << 20  # (all of them: 6.6 GiB)
    assert keys(28, 60, 8, 8192 // 16) == 0
    assert keys(4, 2, 8, 66000 // 16) == 4 * 2 * 8 * 4 * 66000
    for layers, batch, heads, blocks in ((1, 1, 8, 1 << 20), (3, 500, 4, 1 << 17), (200, 3, 1, 1 << 18), (300, 7, 2, 4096)):
        one = heads * blocks * 16 * 4
        assert one <= keys(layers, batch, heads, blocks) <= max(one, 256 << 20)


def test_new_lengths_over_the_old_ones_are_refused(lib):  # noqa: F811
    """The rows move by the old lengths, behind the launch that writes the new ones."""
    assert evict(lib, lens=p, new=p) == -2 and evict(lib, lens=p, new=p + 8) == -2
    assert evict(lib, lens=p + 12, new=p, lens_dt=0) == -2


def test_tables_at_the_end_of_32_bits(lib):  # noqa: F811
    """Token numbers and a grid's stride past them (2^18) are held in 32 bits."""
    def tokens(n):
        return evict(lib, bs=16, blocks=n // 16, stride=n // 16, batch=1, ws_bytes=0)

    assert tokens(2 ** 31 - 2 ** 18) == -2 and tokens(2 ** 31 - 2 ** 16) == -2
    assert tokens(2 ** 31 - 2 ** 20) == -7


def test_trim_refusals(lib):  # noqa: F811
    def trim(bt=p, stride=4, blocks=4, lens=p, held=p, refs=p, pages=10, bs=16, rows=3):
        return lib.mkv_trim_pages(bt, stride, blocks, lens, held, refs, pages, bs, rows, None)

    assert trim(rows=1025) == -2 and trim(rows=-1) == -2 and trim(pages=1 << 31) == -2 and trim(bs=12) == -6
    assert trim(stride=3) == -9 and trim(bt=None) == -1 and trim(lens=None) == -1 and trim(held=None) == -1
    assert trim(refs=None) == -1 and trim(rows=0) == 0


def test_the_wrapper_s_checks():
    kv, w = torch.zeros(4, 16, 2, 8), torch.zeros(4, 16, 2)
    with pytest.raises(ValueError, match="no CPU fallback"):
        mkv.CacheEviction([kv], [kv.clone()], [w])
    with pytest.raises(ValueError, match="every layer needs"):
        mkv.CacheEviction([kv], [], [w])
    with pytest.raises(ValueError, match="every layer needs"):
        mkv.CacheEviction([], [], [])
    with pytest.raises(ValueError, match="go together"):
        mkv.CacheEviction([kv], [kv], [w], [w])
