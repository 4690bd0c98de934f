"""The engine's reports of log probabilities for requests of unlike temperatures:
they are of the model's distribution, whatever the tokens were drawn by."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from mkv import engine as E
from test_gpu_speculative import BS, CFG

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("use_graphs", [True, False])
def test_reports_do_not_depend_on_the_temperature(dev, use_graphs):
    announce(f"engine: reports at temperatures of 0.3 to 4, graphs {use_graphs}")
    g = torch.Generator().manual_seed(23)
    prompts = [torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in (9, 9, 40)]
    model = E.Qwen3Model(CFG, dev, seed=5, block_size=BS)
    eng = E.Engine(model, num_blocks=96, max_num_seqs=4, max_num_batched_tokens=64, max_model_len=256,
                   use_graphs=use_graphs)
    reqs = [eng.add_request(p, 5, temperature=t, logprobs=2) for p, t in zip(prompts, (4.0, 0.3, 2.5))]
    seen = 0
    while not eng.sched.done():
        before = [(r, len(r.reports)) for r in reqs]
        eng.step()
        if not eng.last_sampled:
            continue
        x = torch.log_softmax(eng.last_logits.double(), -1)  # (no temperature)
        entropy = -(x.exp() * x).sum(-1)
        for r, n in before:
            for rep in r.reports[n:]:
                # (the row of the step is the one of this token and entropy)
                rows = [i for i, tok in enumerate(eng.last_sampled) if tok == r.tokens[-1]
                        and abs(float(entropy[i]) - rep.entropy) <= 1e-4]
                assert rows and abs(float(x[rows[0], r.tokens[-1]]) - rep.logprob) <= 1e-5
                assert [t for t, _ in rep.top] == torch.sort(eng.last_logits[rows[0]].float(), descending=True,
                                                             stable=True).indices[:2].tolist()
                seen += 1
    assert seen == 15
