"""Launches of the speculative step's operators whose grids would pass 2^32
threads, refused by their sizes, on the CPU."""
from __future__ import annotations

import ctypes

import pytest

from mkv import _lib
from test_step_operators_host import lib, p, tree  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("kv_dt", [_lib.DTYPE_BF16, _lib.DTYPE_F32])
@pytest.mark.parametrize("blocks", [4, 4096])
def test_tree(lib, kv_dt, blocks):  # noqa: F811
    big = dict(max_blocks=blocks, bt_stride=blocks, kv_dt=kv_dt, q_dt=kv_dt, ws_bytes=1 << 62, total=1 << 22)
    assert tree(lib, seqs=1 << 22, **big) == -2


def test_pages(lib):  # noqa: F811
    ptrs, rows = (ctypes.c_void_p * 64)(*[4096] * 64), (ctypes.c_int64 * 64)(*[1 << 24] * 64)
    pool = [ctypes.addressof(ptrs), ctypes.addressof(rows), 64, 10]
    assert lib.mkv_copy_pages(*pool, 1 << 10, p, p, 1, 3, None) == -2
    odd = (ctypes.c_int64 * 64)(*[(1 << 24) - 4] * 64)
    assert lib.mkv_compact_slots(ctypes.addressof(ptrs), ctypes.addressof(odd), 64, 10, 16, p, 4, 4, p, 1, p, 1, 2048, 2,
                                 2048, None) == -2
    need = lib.mkv_assign_pages_workspace_size(6, 4)
    assert lib.mkv_assign_pages(*pool, 1 << 10, p, 4, 4, p, p, p, p, 1, p, 1, p, 6, p, need, None) == -2
