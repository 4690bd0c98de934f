"""GPU parity of tree attention over per-token-head caches whose V scales are
far from 1 or far from each other, against its definition in float64.

Bounds, for each output by itself.  With A = sum_j p_j |v_j| / sum_j p_j:

* P times the V scale is rounded to fp16 once, half a step of 2^-11 of each
  term: 2^-11 A;
* the fp32 arithmetic as in the tests of usual scales, every part of it relative
  to the terms: 2^-11 A;
* a product below fp16's normal range is off by up to 2^-25 where the row's
  largest is 2^7 or more: 2^-32 of the largest term for each key;
* the store's half step.
"""
from __future__ import annotations

import math

import pytest
import torch

from conftest import announce
from test_gpu_tree import SHAPES, dequantised, make, reference, run

pytestmark = pytest.mark.gpu

FORMATS = ["fp8_token", "int8_token"]
# beside the usual ones: tables that are split, over one, two and four row groups
WIDE = {"split": ([5, 9], [3100, 900], 4, 2, 128, 16), "split64": ([30, 9], [2100, 500], 4, 2, 128, 16),
        "split128": ([70, 9], [1300, 500], 4, 2, 128, 16), "split_d64": ([5, 9], [3100, 900], 4, 2, 64, 16)}


def case(fmt, shape, seed):
    c = make(fmt, *{**SHAPES, **WIDE}[shape], seed=seed)
    c["q"] = c["q"].to(torch.bfloat16)  # (its exponents hold every output here)
    return c


def largest_term(c):
    """max_j p_j |v_j| / sum_j p_j over all rows, at most the largest |v| seen."""
    return float(dequantised(c["v"], c["vs"], c["mode"]).nan_to_num(0, 0, 0).abs().max())


def check(c, dev, times=1.0, top=None):
    """With every V scale `times` what it is (a power of two): `times` the output."""
    got = run(c, dev, vs=c["vs"] * times).double().cpu() / times
    total = int(c["cu"][-1])
    want = reference(c)
    a = reference({**c, "v": c["v"].float().abs(), "vs": c["vs"].abs()})
    keys = int(c["ctx"].max())
    tol = 2.0 ** -10 * a + keys * 2.0 ** -32 * (largest_term(c) if top is None else top)
    tol = tol + torch.where(want == 0, 0.0, 0.5 * torch.exp2(torch.floor(torch.log2(want.abs())) - 7))
    err = (got - want).abs()[:total]
    assert bool((err <= tol[:total]).all()), (
        f"{int((~(err <= tol[:total])).sum())} of {err.numel()} out of tolerance; "
        f"largest error {float(err.nan_to_num(math.inf).max()):.3e}, output {float(want.abs().max()):.3e}")


@pytest.mark.parametrize("power", [-60, -40, -20, -10, 8, 20, 90])
@pytest.mark.parametrize("shape", ["odd_group", "rows64", "rows128", "d64", *WIDE])
@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_of_any_size(dev, fmt, shape, power):
    announce(f"tree {fmt} {shape}, V scales x 2^{power}")
    check(case(fmt, shape, seed=power + 100), dev, times=2.0 ** power)


@pytest.mark.parametrize("shape", ["odd_group", "rows128", "d64", *WIDE])
@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_far_from_each_other(dev, fmt, shape):
    """Neighbouring tokens' V scales 2^-16 to 2^16 times the usual."""
    announce(f"tree {fmt} {shape}, mixed V scales")
    c = case(fmt, shape, seed=5)
    g = torch.Generator().manual_seed(6)
    c["vs"] = c["vs"] * torch.exp2(torch.randint(-16, 17, c["vs"].shape, generator=g).float())
    check(c, dev)


@pytest.mark.parametrize("logit", [9.0, 16.0])
@pytest.mark.parametrize("small", [1e-2, 1e-5, 0.0])
@pytest.mark.parametrize("shape", ["rows64", "d64", "split", "split_d64"])
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_sink(dev, fmt, shape, small, logit):
    """The first token draws most of every row's weight, and its own V scale is
    a hundredth, 10^-5 or none of the others'."""
    announce(f"tree {fmt} {shape}, a sink of logit {logit} with V scale x {small}")
    c = case(fmt, shape, seed=7)
    u = torch.where(torch.arange(c["D"]) % 3 == 0, -1.0, 1.0)
    for s in range(len(c["ctx"])):
        page = int(c["bt"][s, 0])
        c["k"][page, 0] = (u * 16).to(c["k"].dtype)
        c["ks"][page, 0] = 1 / 32  # k = u / 2
        c["vs"][page, 0] *= small
    at = logit / (0.5 * c["D"] * c["scale"])
    c["q"] = (c["q"].float() * 0.2 + at * u).to(torch.bfloat16)
    check(c, dev)


@pytest.mark.parametrize("shape", ["rows64", "d64"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("value", [2.0 ** 60, math.inf, math.nan])
def test_scales_that_no_row_sees(dev, fmt, shape, value):
    """A drafted token that some rows do not see, and slots behind the context,
    may have any V scale: the other rows have theirs."""
    announce(f"tree {fmt} {shape}, V scale {value} where it is not seen")
    c = case(fmt, shape, seed=8)
    n, ctx = int(c["cu"][1]), int(c["ctx"][0])
    top = largest_term(c)
    t = ctx - n + 2
    page, row = int(c["bt"][0, t // c["bs"]]), t % c["bs"]
    c["mask"][:n, 2] = False
    c["vs"][page, row] = value
    if ctx % c["bs"]:
        c["vs"][int(c["bt"][0, ctx // c["bs"]]), ctx % c["bs"]] = value
    check(c, dev, top=top)
