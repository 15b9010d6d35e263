"""sample_tokens: refusals, no GPU."""
from __future__ import annotations

import pytest
import torch

from tilequant_amd import _native as nat
from tilequant_amd.sampling import sample_tokens

FAKE = 1 << 20


def call(**over):
    a = dict(logits=FAKE, ld=1000, dtype=0, rows=2, vocab=1000, u=FAKE, t=None, t0=1.0, k=None, k0=0, p=None, p0=1.0,
             m=None, m0=0.0, out=FAKE, ws=None, ws_elems=0)
    a.update(over)
    return nat.load().tq_sample_tokens(*a.values(), None)


def test_refusals_come_before_any_launch():
    assert call(dtype=3) == -2
    for bad in (dict(rows=-1), dict(vocab=0), dict(vocab=500001, ld=500001), dict(ld=999), dict(logits=None), dict(u=None),
                dict(out=None)):
        assert call(**bad) == -1, bad
    assert call(logits=FAKE + 1) == -3 and call(dtype=2, logits=FAKE + 2) == -3
    need = nat.load().tq_sample_workspace_elems(2, 100000)      # a long row is split and needs its workspace
    assert need > 0 and nat.load().tq_sample_workspace_elems(2, 1000) == 0
    assert call(vocab=100000, ld=100000) == -4 and call(vocab=100000, ld=100000, ws=FAKE, ws_elems=need - 1) == -4
    assert call(rows=0, logits=None, u=None, out=None) == 0


def test_no_cpu_tensors():
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        sample_tokens(torch.zeros((2, 10)), torch.zeros(2))
