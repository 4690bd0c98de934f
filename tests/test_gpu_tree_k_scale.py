"""GPU parity of tree attention over FP8 caches whose per-tensor K scale is zero or
negative, against its definition in float64 (the bounds of usual scales)."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_gpu_tree import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k_scale", [0.0, -0.013])
@pytest.mark.parametrize("D", [128, 64])
def test_k_scales_of_a_caller(dev, k_scale, D):
    """A per-tensor K scale of 0 (every key that is seen weighs the same) and a
    negative one."""
    announce(f"tree fp8 head_dim {D}, K scale {k_scale}")
    for draft, prefix in (([5, 33, 1], [30, 200, 7]), ([70], [90]), ([4], [2100])):
        c = make("fp8", draft, prefix, 8, 4, D, 16, seed=3)
        c["ks"] = torch.tensor([k_scale])
        check(c, dev)
