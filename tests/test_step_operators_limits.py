"""Sizes that the speculative step's operators refuse ahead of any launch, on
the CPU: counts that their 32-bit indexes or grids would not hold."""
from __future__ import annotations

import pytest

from mkv import _lib
from test_step_operators_host import lib, p, tree  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("total,cols,heads", [(1 << 27, 1 << 27, 16), (1 << 30, 1 << 20, 2), (2 ** 31 - 1, 2 ** 31 - 1, 1)])
def test_more_rows_than_the_grid_takes(lib, total, cols, heads):  # noqa: F811
    assert tree(lib, total=total, cols=cols, mask_stride=0, hq=heads, hkv=1) == -2
    assert lib.mkv_paged_tree_workspace_size(2, total, heads, 1, 128, 16, 4, cols, _lib.DTYPE_BF16) == 0


def test_many_rows_that_it_takes(lib):  # noqa: F811
    need = lib.mkv_paged_tree_workspace_size(1, 65000, 16, 1, 128, 16, 4096, 65000, _lib.DTYPE_BF16)
    assert need >= 65000 * 16 * 130 * 4


def test_pages_and_logits(lib):  # noqa: F811
    assert lib.mkv_token_logprobs(p, p, p, p, p, 100, _lib.DTYPE_BF16, 1 << 31, 100, p, 1, 1, 1, 5, p, 1 << 62, None) == -2
    assert lib.mkv_assign_pages_workspace_size(0, 4) == 0
