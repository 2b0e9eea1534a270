"""attn_decode_shared over int8 keys, queries whose values are of very different size: what a large value meets may be
codes of zero, and the small ones then decide.

Where few rows see a prefix, a query is held as a whole number of 24 bits wherever what that leaves out moves no score by more
than 2^-16 (in powers of two), a weight of the softmax hence by at most ln(2) 2^-16 of itself; that joins the
weights' rounding to two bf16 numbers (2^-16, attn_ref.py), twice, as the sum of weights moves too."""
from __future__ import annotations

import math

import attn_ref as R
import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
UP = (1 + 2 * math.log(2)) * 2.0 ** -16


def check(c):
    """Batch.check, with UP; a query head that holds a number that is not finite gives none."""
    b = 0
    for g, (n, p) in enumerate(c.groups):
        kp, vp = R.gathered(c.cache, c.ptable, g, p)
        for _ in range(n):
            ko, vo = R.gathered(c.cache, c.table, b, c.own[b])
            k, v = torch.cat([kp, ko]), torch.cat([vp, vo])
            seen = torch.ones((1, len(k)), dtype=torch.bool, device=k.device)
            ref, tol = R.attend(c.q[b:b + 1], k, v, c.scale, seen, c.dt, UP)
            ok = c.q[b].isfinite().all(-1)
            assert bool(c.out[b, ~ok].isnan().all())
            R.check(c.out[b, ok], ref[0, ok], tol[0, ok], f"sequence {b}")
            b += 1


@pytest.mark.parametrize("times", [1e3, 1e5, 1e7, 1e9, 1e25])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,hq", [(3, 8), (1, 2), (20, 8), (3, 36)])
def test_a_large_value_meets_codes_of_zero(n, hq, hd, times):
    c = S.Batch([(n, 300), (1, 0), (1, 40)], [40 + i for i in range(n + 2)], hq, 2, hd, BF, seed=hd + n, page=16, int8=True)
    c.cache[0][..., 5] = 0
    c.q[..., 5] = times
    c.q[0, 0, 5] = -3 * times
    c.run()
    check(c)


@pytest.mark.parametrize("n", [3, 20])
@pytest.mark.parametrize("hd", [64, 256])
def test_fp16_queries(n, hd):
    """Of fp16's whole range: values of a thousandth beside the largest there are."""
    c = S.Batch([(n, 300)], [40 + i for i in range(n)], 8, 2, hd, F16, seed=hd, page=16, int8=True, scale=300.0 * hd ** -0.5)
    c.q.mul_(2.0 ** -10)
    c.cache[0][..., 5] = 0
    c.q[:, ::2, 5] = 60000.0
    c.run()
    check(c)


@pytest.mark.parametrize("n", [3, 20])
@pytest.mark.parametrize("dt", [BF, F16])
def test_values_of_every_size(n, dt):
    """Sixteen large values of sizes from 2^3 to 2^15 (as fp16 some are infinite), against codes of zero in some sequences' keys and in
    the prefix's; the own keys of one sequence meet them all, and the sequence without them is as ever."""
    hd = 128
    c = S.Batch([(n, 500)], [30] * n, 8, 2, hd, dt, seed=n, page=16, int8=True)
    k = c.cache[0]
    other = c.table[0, :2].long()
    keep = k[other].clone()
    k[..., :16] = 0
    k[other] = keep
    g = torch.Generator(device="cuda").manual_seed(3)
    sizes = 2.0 ** (3 + 12 * torch.arange(16, device="cuda") / 15)
    c.q[1:, :, :16] = (sizes * torch.randn((n - 1, 8, 16), generator=g, device="cuda")).to(dt)
    c.run()
    check(c)


@pytest.mark.parametrize("n", [3, 20])
def test_rows_of_one_value_and_of_powers(n):
    """Rows of a single value that is not zero, of powers of two over bf16's range, and of numbers next to the largest of
    their power."""
    c = S.Batch([(n, 200)], [17] * n, 8, 2, 64, BF, seed=n + 1, page=16, int8=True)
    c.cache[0][..., :32] = 0
    c.q[0, 0] = 0
    c.q[0, 0, 40] = 1.5
    c.q[0, 1, :32] = 2.0 ** torch.linspace(-126, 100, 32, device="cuda").round()
    c.q[0, 2] = (2 - 2.0 ** -7) * torch.sign(c.q[0, 2].float()).to(BF)
    c.q[0, 3] = (2 - 2.0 ** -7) * 2.0 ** -9
    c.q[0, 3, 63] = 2 - 2.0 ** -7
    c.q[1, 0, 40:] *= 2.0 ** -60
    c.q[1, 0, 0] = 2.0 ** -100
    c.run()
    check(c)


def test_other_sequences_keep_their_bits():
    """A sequence of ordinary values beside one of very different ones, and beside ordinary ones: within the allowed
    error of the formula either way."""
    c = S.Batch([(4, 1000)], [30, 31, 32, 33], 8, 2, 128, BF, seed=9, page=16, int8=True)
    c.run()
    check(c)
    c.cache[0][..., 9] = 0
    c.q[2, :, 9] = 1e8
    c.run()
    check(c)


def test_infinite_scales_beside_large_values():
    """A scale that is not finite makes numbers of nothing that sees its key, however the query is held."""
    c = S.Batch([(3, 100)], [20, 21, 22], 8, 2, 128, BF, seed=83, page=16, int8=True)
    c.cache[0][..., 5] = 0
    c.q[0, :, 5] = 1e8
    c.cache[2][c.table[1, 0].long(), 3] = float("-inf")
    c.q[2, 1, 7] = float("nan")
    c.run()
    ref, tol = c.expected()  # (values are at most 127 x 0.022: UP allows 2 ln(2) 2^-16 of that more, below 2^-14)
    assert bool(c.out[1].isnan().all()) and bool(c.out[2, 1].isnan().all())
    R.check(c.out[0], ref[0], tol[0] + 2.0 ** -14)
    ok = [h for h in range(8) if h != 1]
    R.check(c.out[2, ok], ref[2, ok], tol[2, ok] + 2.0 ** -14)
