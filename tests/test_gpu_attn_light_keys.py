"""One key far above very many others, with a value of zero as an attention sink has: the output is of the
others alone, each of whose weights is a small part of the sink's (fp16 has five bits of exponent)."""
from __future__ import annotations

import math

import pytest
import torch

import attn_far as F
import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _inputs(n, hd, at, octaves, dt, seed, rows=1, G=4):
    """Queries of one direction, n keys near it with scores of a deviation of 0.3, the sink at `at`
    `octaves` above them (for the first head; up to a tenth less for others), values around 1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn(hd, generator=g, device="cuda").sign()
    q = (base * (1 - 0.1 * torch.rand((rows, G, 1), generator=g, device="cuda"))).to(dt)
    q[:, 0] = base.to(dt)
    k = (torch.randn((n, 1, hd), generator=g, device="cuda") * 0.3).to(dt)
    v = (1 + 0.25 * torch.randn((n, 1, hd), generator=g, device="cuda")).to(dt)
    k[at, 0] = (base * (octaves * math.log(2) * hd ** -0.5)).to(dt)
    v[at] = 0
    return q, k, v


def _check(out, q, k, v, dt, name):
    """One row [G, hd] against 64 bits."""
    o, tol, _ = F.row(q, k[:, 0], v[:, 0], dt)
    assert (o.abs() > 4 * tol).float().mean() > 0.9, f"{name}: the tolerance does not tell a zero"
    R.check(out, o, tol, name)


def _paged(k, v, page, seed):
    c, table = F.paged(k[:, 0], v[:, 0], page, seed)
    return c[:2], table


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# (at 2^20 keys 30 octaves leave 2^-10 of the weight to the others)
@pytest.mark.parametrize("n,octaves", [(16384, 18), (16384, 23), (131072, 18), (131072, 25.3), ((1 << 20) + 7, 25.3),
                                       ((1 << 20) + 7, 30)])
@pytest.mark.parametrize("where", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("dt", [FP, BF])
def test_decode(n, octaves, where, dt):
    from qwen35_amd.kernels import attention as A
    hd = 64 if n > 200000 else 128
    at = min(int(n * where), n - 1)
    q, k, v = _inputs(n, hd, at, octaves, dt, n + int(octaves))
    (kc, vc), table = _paged(k, v, 256, 3)
    out = torch.empty_like(q)
    A.attn_decode(q, kc, vc, table, _ints(n), out)
    _check(out[0], q[0], k, v, dt, f"sink at {at}")


@pytest.mark.parametrize("octaves", [18, 23])
@pytest.mark.parametrize("dt", [FP, BF])
def test_decode_of_many_sequences(octaves, dt):
    """More sequences than are cut: one workgroup goes over all of a sequence's keys."""
    from qwen35_amd.kernels import attention as A
    n, hd, B = 16384, 64, 1600
    q, k, v = _inputs(n, hd, 40, octaves, dt, octaves, B)
    (kc, vc), table = _paged(k, v, 256, 6)
    out = torch.empty_like(q)
    A.attn_decode(q, kc, vc, table.expand(B, -1), _ints(n).expand(B).contiguous(), out)
    for b in (0, 777, B - 1):
        _check(out[b], q[b], k, v, dt, f"sequence {b}")


@pytest.mark.parametrize("rows", [8, 300])          # halved tiles and whole ones
@pytest.mark.parametrize("hd,n,octaves", [(64, 131072, 25.3), (128, 131072, 22), (256, 40000, 22), (64, (1 << 20) + 7, 28)])
@pytest.mark.parametrize("where", [0.0, 0.6])
@pytest.mark.parametrize("dt", [FP, BF])
def test_a_chunk_over_the_cache(rows, hd, n, octaves, where, dt):
    from qwen35_amd.kernels import attention as A
    at = int(n * where)
    q, k, v = _inputs(n, hd, at, octaves, dt, n + hd, rows)
    (kc, vc), table = _paged(k, v, 128, 4)
    out = torch.empty_like(q)
    A.attn_prompt_paged(q, kc, vc, table, _ints(n), _ints(0, rows), out)
    for i in (0, rows // 2, rows - 1):
        _check(out[i], q[i], k[:n - rows + 1 + i], v[:n - rows + 1 + i], dt, f"row {i}, sink at {at}")


@pytest.mark.parametrize("hd,n,octaves", [(64, 30000, 21), (128, 20000, 20.5), (256, 9000, 19), (256, 700, 15)])
@pytest.mark.parametrize("dt", [FP, BF])
def test_a_prompt(hd, n, octaves, dt):
    """The first key is the sink, as in a prompt that starts with one."""
    from qwen35_amd.kernels import attention as A
    q, k, v = _inputs(n, hd, 0, octaves, dt, n, n)
    out = torch.empty_like(q)
    A.attn_prompt(q, k, v, _ints(0, n), out)
    for i in (n // 4, n // 2, n - 30, n - 1):
        _check(out[i], q[i], k[:i + 1], v[:i + 1], dt, f"row {i}")


@pytest.mark.parametrize("dt", [FP, BF])
def test_scores_that_rise_and_fall_by_many_octaves(dt):
    """Runs of keys up and down 40 octaves: the reference goes with them both ways, and the sums are those
    of the heaviest."""
    from qwen35_amd.kernels import attention as A
    n, hd, rows = 3000, 128, 40
    q, k, v = _inputs(n, hd, 5, 1, dt, 7, rows)
    base = q[0, 0].float()
    wave = torch.sin(torch.arange(n, device="cuda") / 150.0) * 20 * math.log(2) * hd ** -0.5
    k[:, 0] = (k[:, 0].float() + base * wave[:, None]).to(dt)
    (kc, vc), table = _paged(k, v, 64, 5)
    out, packed, one = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q[:1])
    A.attn_prompt_paged(q, kc, vc, table, _ints(n), _ints(0, rows), out)
    A.attn_prompt(q, k, v, _ints(0, rows), packed, cu_k=_ints(0, n))
    A.attn_decode(q[rows - 1:], kc, vc, table, _ints(n), one)
    for i in (0, rows - 1):
        for y in (out, packed):
            _check(y[i], q[i], k[:n - rows + 1 + i], v[:n - rows + 1 + i], dt, f"row {i}")
    _check(one[0], q[rows - 1], k, v, dt, "decode")
