"""What the verification of drafted tokens refuses, on the CPU: the wrapper's
checks and the library's own (which return before any launch)."""
from __future__ import annotations

import pytest
import torch

import mkv
from mkv import _lib
from test_step_operators_host import lib, p  # noqa: F401  (lib: a fixture)


def verify(lib, **over):  # noqa: F811
    a = dict(acc=p, num=p, nxt=p, chance=p, logits=p, stride=100, draft=p, draft_stride=100, dt=_lib.DTYPE_BF16, total=6,
             vocab=100, ids=p, ids_dt=1, parents=p, par_dt=1, cu=p, seqs=2, nodes=4, u=p, noise=p, noise_stride=100,
             temps=p, ws=p, ws_bytes=1 << 20, stream=None)
    assert set(over) <= set(a)
    a.update(over)
    return lib.mkv_verify_drafts(*a.values())


def test_refusals(lib):  # noqa: F811
    assert verify(lib, vocab=0) == -2 and verify(lib, total=-1) == -2 and verify(lib, seqs=-1) == -2
    assert verify(lib, seqs=70000) == -2 and verify(lib, nodes=0) == -2 and verify(lib, nodes=1025) == -2
    assert verify(lib, dt=_lib.DTYPE_I8) == -3 and verify(lib, ids_dt=4) == -3 and verify(lib, par_dt=4) == -3
    for name in ("acc", "num", "nxt", "chance", "logits", "ids", "cu", "u", "noise", "ws"):
        assert verify(lib, **{name: None}) == -1, name
    assert verify(lib, stride=99) == -9 and verify(lib, draft_stride=99) == -9 and verify(lib, noise_stride=99) == -9
    assert verify(lib, logits=p + 1) == -8 and verify(lib, draft=p + 1) == -8 and verify(lib, noise=p + 2) == -8
    assert verify(lib, ws=p + 8) == -8
    need = lib.mkv_verify_drafts_workspace_size(6, 100, 2, 4, 1)
    assert need > lib.mkv_verify_drafts_workspace_size(6, 100, 2, 4, 0) > 0 and verify(lib, ws_bytes=need - 1) == -7
    assert verify(lib, seqs=0) == 0
    assert lib.mkv_verify_drafts_workspace_size(6, 100, 2, 1025, 1) == 0
    # (a grid past 2^32 threads)
    big = 0x7fff0000
    assert verify(lib, vocab=big, stride=big, draft_stride=big, noise_stride=big, seqs=1000, ws_bytes=1 << 62) == -2


def test_the_wrapper_s_checks():
    x = torch.zeros(4, 9)
    ids, cu, u, e = torch.zeros(4, dtype=torch.int64), torch.tensor([0, 4]), torch.zeros(4), torch.ones(1, 9)
    with pytest.raises(ValueError, match="no CPU fallback"):
        mkv.verify_drafts(x, ids, cu, u, e, 4)
