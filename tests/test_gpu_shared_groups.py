"""attn_decode_shared of many small groups: their sums lie next to each other in the workspace, whatever a tile could hold."""
from __future__ import annotations

import random

import attn_ref as R
import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def check_some(c, some):
    starts = [sum(n for n, _ in c.groups[:g]) for g in range(len(c.groups) + 1)]
    up = 2.0 ** -16 if c.cache[2] is not None else None
    for b in some:
        g = max(i for i, s in enumerate(starts[:-1]) if s <= b and starts[i + 1] > b)
        (kp, vp), (ko, vo) = R.gathered(c.cache, c.ptable, g, c.groups[g][1]), R.gathered(c.cache, c.table, b, c.own[b])
        k, v = torch.cat([kp, ko]), torch.cat([vp, vo])
        seen = torch.ones((1, len(k)), dtype=torch.bool, device=k.device)
        R.check(c.out[b:b + 1], *R.attend(c.q[b:b + 1], k, v, c.scale, seen, c.dt, up), f"sequence {b}")


@pytest.mark.parametrize("hq,hkv,hd,n", [(16, 16, 256, 1024), (64, 2, 128, 700), (3, 1, 64, 5000)])
@pytest.mark.parametrize("int8", [False, True])
def test_a_group_of_each_sequence(hq, hkv, hd, n, int8):
    rng = random.Random(n)
    groups = [(1, rng.choice([0, 1, 40, 70])) for _ in range(n)]
    own = [rng.choice([0, 1, 17, 33]) for _ in range(n)]
    groups[n // 2], own[n // 3] = (1, 9000), 5000
    c = S.Batch(groups, own, hq, hkv, hd, BF, seed=n, page=16, int8=int8, pad=1)
    c.run()
    check_some(c, [0, 1, 63, 64, n // 3, n // 2, n - 1, *rng.sample(range(n), 30)])
    assert bool((c.out[-1] == 7.0).all())
    first = c.out.clone()
    c.out.fill_(0.0)
    c.run()
    assert torch.equal(c.out[:-1], first[:-1])


@pytest.mark.parametrize("hq,hkv,hd,int8", [(8, 2, 128, False), (8, 2, 256, True), (40, 2, 64, False), (4, 4, 128, True)])
def test_one_large_group_among_small_ones(hq, hkv, hd, int8):
    """Groups of one sequence on either side of one of 90; prefixes cut into many parts and into one."""
    groups = [(1, 300)] * 70 + [(90, 4000)] + [(0, 800)] + [(1, 33)] * 3 + [(2, 2000)] + [(1, 0)] * 2
    n = sum(m for m, _ in groups)
    c = S.Batch(groups, [(i * 7) % 50 for i in range(n)], hq, hkv, hd, F16, seed=hd, page=16, int8=int8)
    c.run()
    check_some(c, [0, 63, 69, 70, 71, 85, 86, 101, 102, 158, 159, 160, 161, 162, 163, 164, n - 1])


def test_few_cuts():
    """A call near the most that a workspace holds is cut into a few long units; a graph of it replays."""
    from qwen35_amd.kernels import qlin as C
    n, hq, hkv, hd = 1900, 32, 8, 256
    groups = [(1900 // 19, 100 + i) for i in range(19)]
    c = S.Batch(groups, [i % 40 for i in range(n)], hq, hkv, hd, BF, seed=5, page=16)
    c.run()
    check_some(c, [0, 99, 100, 950, 1000, n - 1])
    want = c.out.clone()
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        c.run()
    for _ in range(3):
        c.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, want)
        c.run()
