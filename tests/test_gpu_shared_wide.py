"""attn_decode_shared with more rows of a key head than a tile of 16 has: head groups that do not divide a tile, and what a
device may find in tables, values and scores, there too."""
from __future__ import annotations

import attn_ref as R
import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("hq,hkv,n", [(3, 1, 43), (5, 1, 30), (10, 2, 13), (7, 1, 19), (17, 1, 3), (34, 2, 9), (64, 1, 5), (1, 1, 130),
                                      (12, 4, 100), (63, 1, 2), (11, 1, 2)])
@pytest.mark.parametrize("hd,dt,int8", [(64, BF, True), (128, F16, False), (128, BF, True), (256, BF, False), (256, F16, True)])
def test_heads_that_do_not_divide_a_tile(hq, hkv, n, hd, dt, int8):
    m = max(1, n // 3)
    c = S.Batch([(n, 333), (m, 65), (m, 0)], [(7 * i) % 70 for i in range(n + 2 * m)], hq, hkv, hd, dt, seed=n + hq, page=16,
                int8=int8, pad=2)
    c.run()
    c.check(c.out)
    assert bool((c.out[-2:] == 7.0).all())


@pytest.mark.parametrize("int8", [False, True])
def test_bad_pages(int8):
    """A page outside the cache in a prefix of many rows makes all that see it none, and nothing else; one behind the
    prefix's end is never looked at."""
    n = 40
    c = S.Batch([(n, 90), (n, 200)], [5] * (2 * n), 8, 2, 128, BF, seed=11, page=16, int8=int8)
    ref, tol = c.expected()
    c.ptable[1, 7] = 1 << 30
    c.ptable[0, 6:] = -1
    c.run()
    assert bool(c.out[n:].isnan().all())
    R.check(c.out[:n], ref[:n], tol[:n])


def test_light_keys_beside_a_heavy_one():
    """fp16: as few rows do, many keep the weight of keys 24 octaves lighter than another block's one."""
    page, hd, n = 64, 64, 40
    c = S.Batch([(n, 8192)], [100] * n, 1, 1, hd, F16, seed=53, page=page, scale=1.0)
    k, v, _, _ = c.cache
    k.zero_(), v.zero_(), c.q.zero_()
    c.q[:, :, 0] = 1.0
    k[c.ptable[0, 0].long(), 0, 0, 0] = 17.0                 # 24.5 octaves above the others
    for t, m in ((c.ptable[0], 8192), *((c.table[b], 100) for b in range(n))):
        v[t[:-(-m // page)].long(), :, 0, 1] = 30000.0
    # the heavy key's own block stays out (a key more than 6 octaves lighter than its own block's heaviest loses
    # precision): its other keys and values are nothing
    v[c.ptable[0, 0].long(), :, 0, 1] = 0.0
    c.run()
    c.check(c.out)


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("int8", [False, True])
def test_scores_of_a_large_deviation(dt, int8):
    n = 33
    c = S.Batch([(n, 1500)], [(11 * i) % 90 for i in range(n)], 8, 2, 128, dt, seed=59, page=16, scale=0.5, int8=int8)
    c.run()
    c.check(c.out)


@pytest.mark.parametrize("int8", [False, True])
def test_same_bits_whatever_ran_before(int8):
    """The same call again, after others of other sizes on the same workspace, gives the same bits."""
    c = S.Batch([(50, 3000), (4, 100)], [33] * 54, 16, 2, 128, BF, seed=61, page=32, int8=int8)
    c.run()
    want = c.out.clone()
    for other in (S.Batch([(3, 200)], [9] * 3, 8, 2, 256, BF, seed=62), S.Batch([(70, 100)], [3] * 70, 4, 4, 64, F16, seed=63)):
        other.run()
        c.out.zero_()
        c.run()
        assert torch.equal(c.out, want)
