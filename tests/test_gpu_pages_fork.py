"""PagePool.fork over any iterable of rows."""
from __future__ import annotations

import pytest
import torch

import mkv
from conftest import announce
from test_gpu_pages import caches

pytestmark = pytest.mark.gpu


def test_fork_takes_any_iterable(dev):
    announce("fork, rows by an iterator")
    ts = caches(dev, 20, 16, [(torch.float32, (1,))])
    pool = mkv.PagePool(torch.zeros(4, 8, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.int64, device=dev),
                        mkv.CachePages(ts))
    pool.assign(torch.tensor([0, -1, -1, -1], device=dev), torch.tensor([40, 0, 0, 0], device=dev))
    pool.seq_lens[0] = 40
    assert pool.fork(0, iter([1, 3])).all()
    assert pool.seq_lens.tolist() == [40, 40, 0, 40]
    with pytest.raises(ValueError, match="not among"):
        pool.fork(1, iter([0, 1]))
