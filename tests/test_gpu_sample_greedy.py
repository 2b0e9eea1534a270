"""sample at temperature 0: the largest logit, of equal ones the lowest index, whatever is drawn with."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = (0.0, 0.5, 1 - 2.0 ** -24)


def run(x, u, **kw):
    from qwen35_amd.kernels import sampling
    tokens, lp = torch.full((len(x),), 99, device="cuda"), torch.full((len(x),), 99.0, device="cuda")
    sampling.sample(x.cuda(), torch.full((len(x),), u, device="cuda"), tokens, logprobs=lp, **kw)
    return tokens.cpu(), lp.cpu()


def tied(V, dt):
    """Rows whose largest value is there several times: next to each other, at both ends, in parts of a row that
    different workgroups read, everywhere, as 0 and -0."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn((6, V), generator=g) * 2).clamp(-8, 8).to(dt)
    spread = sorted(torch.randperm(V, generator=g)[:40].tolist())
    x[0, V // 2:V // 2 + 3] = 9.0
    x[1, 0] = x[1, -1] = 9.0
    x[2, spread] = 9.0
    x[3] = -1.5
    x[4] = -x[4].abs() - 1
    x[4, V // 3], x[4, V // 3 + 1], x[4, -1] = -0.0, 0.0, 0.0
    x[5] = -math.inf
    x[5, V // 2:] = torch.finfo(dt).min
    return x, torch.tensor([V // 2, 0, spread[0], 0, V // 3, V // 2])


@pytest.mark.parametrize("V", [300, 8192, 50021, 248320])
@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_the_first_of_equal_ones(V, dt, k):
    x, want = tied(V, dt)
    zeros = torch.zeros(6, device="cuda")
    for u in U:
        for t in (0.0, zeros, zeros - 1):
            tok, _ = run(x, u, top_k=k, temperature=t)
            assert torch.equal(tok, want), (u, t)
            tok, _ = run(x, u, top_k=k, temperature=t, top_p=2.0)
            assert torch.equal(tok, want), (u, t)


def test_rows_that_are_greedy_beside_rows_that_are_not():
    x, want = tied(30000, BF)
    t = torch.tensor([0.0, 1.0, 0.0, 1.0, 0.0, 1.0], device="cuda")
    tok, lp = run(x, 1 - 2.0 ** -24, top_k=128, temperature=t)
    assert torch.equal(tok[::2], want[::2]) and not bool((tok[1::2] == want[1::2]).any())
    same, lp2 = run(x, 1 - 2.0 ** -24, top_k=128, temperature=1.0)
    assert torch.equal(tok[1::2], same[1::2]) and torch.equal(lp[1::2], lp2[1::2])


def test_log_probability_of_a_tie():
    """That of the row as it is: a half for two of one value beside nothing."""
    x = torch.full((1, 20000), -math.inf)
    x[0, [77, 15000]] = 3.0
    for u in U:
        tok, lp = run(x, u, temperature=0.0)
        assert int(tok) == 77 and abs(float(lp) + math.log(2)) <= 2.0 ** -23


def test_infinite_temperature():
    """Infinitely hot rows: all of the k largest weigh the same; where some are infinite only those do, as at any
    temperature."""
    x = -torch.arange(9000.0)[None].repeat(4, 1)
    x[1, [70, 8500]] = math.inf
    x[2, [3, 4, 8999]] = math.inf
    x[3, 1:] = -math.inf
    t = torch.full((4,), math.inf, device="cuda")
    for u, want in ((0.0, [0, 70, 3, 0]), (0.3, [3, 70, 3, 0]), (0.6, [6, 8500, 4, 0]), (0.99, [9, 8500, 8999, 0])):
        tok, _ = run(x, u, top_k=10, temperature=t)
        assert tok.tolist() == want, (u, tok.tolist())
