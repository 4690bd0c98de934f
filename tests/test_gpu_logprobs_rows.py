"""Log probabilities of more rows than a grid's first dimension holds (2^32
threads), against torch in float64."""
from __future__ import annotations

import pytest
import torch

import mkv
from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,top", [(2 ** 26 + 3, 2, 0), (2 ** 25, 5, 1), (2 ** 26 - 1, 1, 1), (2 ** 26 + 1000, 3, 2)])
def test_rows_past_the_grid(dev, rows, vocab, top):
    announce(f"logprobs, {rows} rows of {vocab}, top {top}")
    g = torch.Generator(device=dev).manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device=dev, dtype=torch.bfloat16)
    ids = torch.randint(vocab, (rows,), generator=g, device=dev, dtype=torch.int32)
    got = mkv.token_logprobs(x, ids, top)
    for at in range(0, rows, 1 << 23):
        s = slice(at, min(at + (1 << 23), rows))
        ref = torch.log_softmax(x[s].double(), -1)
        # fp32 arithmetic on a few values of up to 2^3 (as for small vocabularies)
        assert float((got.logprobs[s].double() - ref.gather(1, ids[s].long()[:, None])[:, 0]).abs().max()) <= 1e-5
        assert float((got.entropy[s].double() + (ref.exp() * ref).sum(-1)).abs().max()) <= 4e-5
        if top:
            order = torch.sort(x[s].float(), dim=-1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(got.top_indices[s], order)
            assert float((got.top_logprobs[s].double() - ref.gather(1, order)).abs().max()) <= 1e-5
