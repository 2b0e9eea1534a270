"""attn_decode_shared, fp16: a key as far as 18 octaves below its block's heaviest keeps its weight, however many rows see it
and however heavy other blocks are."""
from __future__ import annotations

import math

import attn_ref as R
import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("block,light", [(0.0, 17.0), (4.0, 17.0), (9.0, 12.0), (15.0, 12.0), (15.5, 17.5), (18.0, 8.0)])
def test_light_keys_beside_their_blocks_heaviest(n, hd, int8, block, light):
    """The first key outweighs the heaviest of each other block of 32 by `block` octaves, and those the other keys of
    their block by `light`; only these have a value in the looked at column."""
    page, length = 64, 4096
    c = S.Batch([(n, length)], [0] * n, 1, 1, hd, F16, seed=53, page=page, scale=1.0, int8=int8)
    k, v, ks, vs = c.cache
    k.zero_(), v.zero_(), c.q.zero_()
    c.q[:, :, 0] = 1.0
    x = torch.full((length,), -(block + light) * math.log(2))
    x[::32] = -block * math.log(2)
    x[0] = 0.0
    y = torch.full((length,), 30000.0)
    y[::32] = 0.0
    ids = c.ptable[0, :length // page].long()
    x, y = (t.cuda().view(-1, page) for t in (x, y))
    if int8:  # (one code, the scales say the rest)
        k[ids, :, 0, 0], v[ids, :, 0, 1] = 100, 100
        ks[ids, :, 0], vs[ids, :, 0] = x / 100, y / 100
    else:
        k[ids, :, 0, 0], v[ids, :, 0, 1] = x.half(), y.half()
    c.run()
    ref, tol = c.expected()
    assert float(ref[0, 0, 1]) > 0.01
    R.check(c.out, ref, tol)
