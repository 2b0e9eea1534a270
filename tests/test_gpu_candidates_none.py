"""Calls of a step of several candidates over a batch of no rows: nothing is done and nothing refused, whatever form their
numbers have."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("history", [0, 7])
@pytest.mark.parametrize("vectors", [False, True])
def test_logits_process(history, vectors):
    from qwen35_amd.kernels import sampling
    e = lambda *s, dt=torch.float32: torch.empty((0, *s), dtype=dt, device="cuda")
    i = lambda *s: e(*s, dt=torch.int32)
    kw = dict(repetition=e(), presence=e(), frequency=e()) if vectors else dict(repetition=1.1, presence=0.5, frequency=0.25)
    out = e(10)
    assert sampling.logits_process(e(10), out, tokens=i(history), lens=i(), prompt_lens=i(), bias_ids=i(3), bias=e(3),
                                   mask=i(1), **kw) is out


@pytest.mark.parametrize("vectors", [False, True])
def test_sample(vectors):
    from qwen35_amd.kernels import sampling
    e = lambda *s, dt=torch.float32: torch.empty((0, *s), dtype=dt, device="cuda")
    kw = dict(temperature=e(), top_p=e(), min_p=e()) if vectors else {}
    tokens = e(dt=torch.int64)
    assert sampling.sample(e(10), e(), tokens, logprobs=e(), **kw) is tokens
