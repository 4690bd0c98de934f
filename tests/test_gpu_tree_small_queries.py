"""GPU parity of tree attention over 1-byte caches with queries near zero, against
its definition in float64 (the bounds of usual ones: no score is off by more)."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_gpu_tree import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["fp8", "fp8_token", "int8_token"])
@pytest.mark.parametrize("size", [1e-20, 1e-37, 1e-39])
def test_queries_near_zero(dev, fmt, size):
    """Rows of q at 10^-20 to 10^-39 beside ordinary ones: every key that they
    see weighs the same, and nothing leaves the operands' range."""
    announce(f"tree {fmt}, rows of q at {size}")
    c = make(fmt, [6, 9], [50, 1300], 8, 4, 128, 16, seed=4)
    c["q"] = c["q"].float()
    c["q"][::2] *= size
    c["q"][1, 3] *= size
    c["q"] = c["q"].to(torch.bfloat16)
    assert bool((c["q"][::2] != 0).any())
    check(c, dev)
    if fmt == "fp8":
        c["scale"] = -c["scale"]
        check(c, dev)
