"""GPU tests of the log probabilities of small vocabularies, which one
workgroup holds (vocabularies of up to 505, 2041 and 8185 logits take unlike
ones; a row's start moves those borders by up to 7), against float64."""
from __future__ import annotations

import pytest
import torch

import mkv
from conftest import announce

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# fp32 arithmetic on values up to 2^6: the sum's and its logarithm's roundings,
# below 8192 terms deep by halves, and the difference's
TOL = 1e-5


def _check(x, ids, top):
    got = mkv.token_logprobs(x, ids, top)
    ref = torch.log_softmax(x.double(), -1)
    want = ref.gather(1, ids.long())
    assert float((got.logprobs.double() - want).abs().max()) <= TOL
    p = torch.where(ref > -torch.inf, ref.exp() * ref, 0.0)
    assert float((got.entropy.double() + p.sum(-1)).abs().max()) <= 4 * TOL
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_indices, order)
    lp = ref.gather(1, order)
    finite = lp > -torch.inf
    assert torch.equal(torch.isinf(got.top_logprobs), ~finite)
    assert float(torch.where(finite, got.top_logprobs.double() - lp, 0.0).abs().max() if top else 0.0) <= TOL


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 504, 505, 506, 511, 513, 2040, 2041, 2042, 2047, 2049, 4095,
                                   8184, 8185, 8186, 8191])
def test_vocabularies_about_the_borders(dev, dtype, vocab):
    announce(f"logprobs, small vocabulary {vocab}, {dtype}")
    g = torch.Generator(device=dev).manual_seed(vocab)
    for top in sorted({0, 1, min(5, vocab), min(64, vocab)}):
        x = (torch.randn(9, vocab, generator=g, device=dev) * 4).to(dtype)
        _check(x, torch.randint(vocab, (9, 3), generator=g, device=dev), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [200, 1500, 8000])
def test_equal_logits_and_masks(dev, dtype, vocab):
    """Many equal logits around the k-th, whole rows of one value, masked
    (-inf) logits in the top, zeros of both signs."""
    announce(f"logprobs, equal logits, vocabulary {vocab}, {dtype}")
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randint(-3, 4, (8, vocab), generator=g, device=dev).to(dtype)
    x[1] = 2.5
    x[2] = torch.where(torch.rand(vocab, generator=g, device=dev) < 0.5, 0.0, -0.0)
    x[3] = -torch.inf
    x[3, torch.randperm(vocab, generator=g, device=dev)[:11]] = 1.0
    x[4, : vocab // 2] = -torch.inf
    x[5, -1], x[6, 0] = 60.0, 60.0
    ids = torch.stack([torch.zeros(8), torch.full((8,), vocab - 1)], 1).long().to(dev)
    ids[3] = x[3].float().argmax()
    ids[4] = vocab - 1
    for top in (1, 7, 40, 64):
        _check(x, ids, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 2000, 8100])
def test_rows_at_any_start_and_the_memory_between_them(dev, dtype, vocab):
    announce(f"logprobs, rows at unlike starts, vocabulary {vocab}, {dtype}")
    g = torch.Generator(device=dev).manual_seed(8)
    buf = torch.full((5, vocab + 9), torch.inf, device=dev, dtype=dtype)
    view = buf[:, 3:3 + vocab]
    view.copy_((torch.randn(5, vocab, generator=g, device=dev) * 4).to(dtype))
    assert vocab + 9 != vocab and view.stride(0) == vocab + 9
    _check(view, torch.randint(vocab, (5, 2), generator=g, device=dev), 20)


@pytest.mark.parametrize("vocab", [100, 1000, 5000])
def test_not_finite_absent_and_outside(dev, vocab):
    announce(f"logprobs, not finite, vocabulary {vocab}")
    x = torch.linspace(-2, 2, 6 * vocab, device=dev).reshape(6, vocab).contiguous()
    x[0, 5] = torch.nan
    x[1, 7] = torch.inf
    x[2] = -torch.inf
    ids = torch.tensor([[3, -1, vocab, 2 ** 40]] * 6, device=dev)
    r = mkv.token_logprobs(x, ids, 4)
    assert torch.isnan(r.logprobs[:3, 0]).all() and torch.isfinite(r.logprobs[3:, 0]).all()
    assert (r.logprobs[:, 1] == 0).all() and torch.isnan(r.logprobs[:, 2:]).all()
    assert torch.isnan(r.entropy[:3]).all() and torch.isfinite(r.entropy[3:]).all()
    assert r.top_indices[0, 0] == 5 and r.top_indices[1, 0] == 7
    assert r.top_indices[2].tolist() == [0, 1, 2, 3]
    many = torch.full((6, 700), 1, device=dev, dtype=torch.int32)  # more tokens than threads
    many[:, 1::2] = vocab - 1
    got = mkv.token_logprobs(x[3:], many[3:], 0).logprobs
    assert torch.equal(got[:, 0::2], got[:, :1].expand(-1, 350)) and torch.equal(got[:, 1::2], got[:, 1:2].expand(-1, 350))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [257, 300, 505, 2041, 8185])
def test_rows_of_one_value_or_two(dev, dtype, vocab):
    """More equal logits than are ranked against each other, in every form."""
    announce(f"logprobs, one value, vocabulary {vocab}, {dtype}")
    x = torch.full((4, vocab), -1.5, device=dev, dtype=dtype)
    x[1, ::2] = 3.0
    x[2, 5:9] = 3.0
    x[3] = -torch.inf
    x[3, vocab - 70:] = 0.25
    ids = torch.full((4, 1), vocab - 1, device=dev)
    for top in (1, 3, 5, 64):
        _check(x, ids, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [400, 2000, 8000, 50257])
def test_the_largest_logits_side_by_side(dev, dtype, vocab):
    """Rows whose largest logits lie in few threads' shares: sorted both ways, a
    run of 300 larger ones (of one value or of many), and larger ones 8192 apart."""
    announce(f"logprobs, large logits together, vocabulary {vocab}, {dtype}")
    g = torch.Generator(device=dev).manual_seed(11)
    x = torch.randn(6, vocab, generator=g, device=dev)
    x[0], x[1] = x[0].sort().values, x[1].sort(descending=True).values
    x[2, 40:340] += 12
    x[3, vocab - 301:vocab - 1] = 9.0
    x[4, ::8] += 12
    x[5, torch.arange(0, vocab, 8192, device=dev)] += 20
    x = x.to(dtype)
    for top in (1, 20, 33, 64):
        _check(x, torch.randint(vocab, (6, 2), generator=g, device=dev), top)
