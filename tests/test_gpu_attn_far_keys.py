"""Very long contexts in which every part counts: each run of 1024 keys holds one key of half the run's
weight, whose value stands in a column of its own (of hd), so that a column's output is the sum of a few known
keys and one run left out or taken twice is far outside the tolerance."""
from __future__ import annotations

import math

import pytest
import torch

import attn_far as F
import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
RUN = 1024


def _inputs(n, hd, rows, G, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn(hd, generator=g, device="cuda").sign()
    q = (base * (1 - 0.02 * torch.rand((rows, G, 1), generator=g, device="cuda"))).to(dt)
    k = (torch.randn((n, hd), generator=g, device="cuda") * 0.3).to(dt)
    v = torch.randn((n, hd), generator=g, device="cuda").to(dt) * 0.25
    runs = -(-n // RUN)
    u = torch.arange(runs, device="cuda")
    # at a run's first key, its last, or anywhere; the last run's at the last key
    off = torch.where(u % 3 == 0, 0, torch.where(u % 3 == 1, RUN - 1, torch.randint(0, RUN, (runs,), generator=g, device="cuda")))
    at = (u * RUN + off).clamp_max(n - 1)
    at[-1] = n - 1
    k[at] = (base * (math.log(RUN) * hd ** -0.5)).to(dt)
    v[at] = 0
    v[at, u % hd] = 64
    return q, k, v, at


def _check(out, q, k, v, at, dt, name, up=None, adds=F.ADDS):
    """One row; `at`: the planted keys that it sees."""
    o, tol, w = F.row(q, k, v, dt, up, adds)
    cols = torch.arange(len(at), device="cuda") % k.shape[1]
    # leaving any planted key out, or a zero in a column that has one, would show
    assert (w[:, at] * 64 > 2 * tol[:, cols]).all(), f"{name}: the tolerance does not tell a run left out"
    assert (o[:, cols].abs() > 8 * tol[:, cols]).all(), name
    R.check(out, o, tol, name)


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["bf16", "fp16", "int8"])
def test_a_million_keys(kind):
    from qwen35_amd.kernels import attention as A
    n, hd, rows, int8 = (1 << 20) + 7, 64, 20, kind == "int8"
    dt = FP if kind == "fp16" else BF
    q, k, v, at = _inputs(n, hd, rows, 4, dt, 1)
    c, table = F.paged(k, v, 256, 2, int8)
    if int8:
        k, v = (x[:, 0] for x in R.gathered(c, table, 0, n))
    out, one = torch.empty_like(q), torch.empty_like(q[:1])
    A.attn_prompt_paged(q, c[0], c[1], table, _ints(n), _ints(0, rows), out, k_s=c[2], v_s=c[3])
    A.attn_decode(q[-1:], c[0], c[1], table, _ints(n), one, k_s=c[2], v_s=c[3])
    for i in (0, 9, rows - 1):
        m = n - rows + 1 + i
        _check(out[i], q[i], k[:m], v[:m], at[at < m], dt, f"row {i}")
    _check(one[0], q[-1], k, v, at, dt, "decode", 2.0 ** -16 if int8 else None)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "int8"])
@pytest.mark.parametrize("hd,rows,n", [(256, 600, 60000), (128, 3, 200001)])
def test_chunks_and_steps_over_long_contexts(kind, hd, rows, n):
    """Whole tiles and halved ones, cut into parts."""
    from qwen35_amd.kernels import attention as A
    int8, dt = kind == "int8", FP if kind == "fp16" else BF
    q, k, v, at = _inputs(n, hd, rows, 4, dt, hd)
    c, table = F.paged(k, v, 64, 3, int8)
    if int8:
        k, v = (x[:, 0] for x in R.gathered(c, table, 0, n))
    out, one = torch.empty_like(q), torch.empty_like(q[:1])
    A.attn_prompt_paged(q, c[0], c[1], table, _ints(n), _ints(0, rows), out, k_s=c[2], v_s=c[3])
    A.attn_decode(q[-1:], c[0], c[1], table, _ints(n), one, k_s=c[2], v_s=c[3])
    for i in (0, rows // 2, rows - 1):
        m = n - rows + 1 + i
        _check(out[i], q[i], k[:m], v[:m], at[at < m], dt, f"row {i}")
    _check(one[0], q[-1], k, v, at, dt, "decode", 2.0 ** -16 if int8 else None)


@pytest.mark.parametrize("hd,T,dt", [(64, 100003, BF), (256, 40001, FP), (128, 9000, BF)])
def test_a_long_prompt(hd, T, dt):
    """Its last rows over all of it (a tile that is not cut adds T / 32 blocks), and rows on the way."""
    from qwen35_amd.kernels import attention as A
    q, k, v, at = _inputs(T, hd, T, 2, dt, T)
    out = torch.empty_like(q)
    A.attn_prompt(q, k[:, None], v[:, None], _ints(0, T), out)
    for i in (5000, T // 2, T - 33, T - 2, T - 1):
        _check(out[i], q[i], k[:i + 1], v[:i + 1], at[at <= i], dt, f"row {i}", adds=32 + (i + 32) // 32)
