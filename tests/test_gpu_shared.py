"""attn_decode_shared against the formula in 64 bits (candidates_ref.py, attn_ref.py)."""
from __future__ import annotations

import random

import attn_ref as R
import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def _own(groups, most, seed):
    rng = random.Random(seed)
    return [rng.choice([0, 1, most, rng.randint(0, most)]) for _ in range(sum(n for n, _ in groups))]


GROUPS = {
    "one": [(1, 1)],
    "few": [(4, 180)],
    "none": [(3, 0)],
    "mixed": [(3, 0), (0, 50), (5, 33), (1, 16), (2, 1000), (0, 0), (7, 31)],
    "most": [(8, 8000)],
    "many": [(40, 700)],
    "lots": [(1, n) for n in range(70)] + [(2, 129)] * 3,
}


@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 1), (12, 4), (1, 1)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("groups", ["one", "few", "none", "mixed"])
def test_groups(groups, int8, dt, hd, hq, hkv):
    g = GROUPS[groups]
    c = S.Batch(g, _own(g, 70, 3), hq, hkv, hd, dt, seed=hd + hq, page=16 if hq == 3 else 64, int8=int8, pad=2,
                head_major=hkv != 4)
    c.run()
    c.check(c.out)
    assert bool((c.out[len(c.own):] == 7.0).all())


@pytest.mark.parametrize("groups,hq,hkv,hd,dt,int8,own", [
    ("most", 8, 2, 256, BF, False, 190), ("most", 8, 2, 256, BF, True, 300), ("many", 8, 2, 256, BF, False, 64),
    ("many", 8, 1, 128, F16, False, 500), ("many", 16, 1, 64, BF, True, 33), ("many", 32, 1, 256, F16, True, 5),
    ("lots", 6, 2, 128, BF, False, 40), ("lots", 4, 4, 64, F16, True, 9), ("many", 64, 1, 128, BF, False, 100),
    ("mixed", 40, 2, 256, F16, False, 100), ("mixed", 34, 2, 64, BF, True, 100), ("few", 16, 1, 128, F16, True, 2000),
    ("few", 7, 1, 256, BF, False, 3333), ("most", 5, 5, 128, F16, False, 1),
])
def test_sizes(groups, hq, hkv, hd, dt, int8, own):
    """Many rows of a key head, long prefixes, long answers, more groups than a wave has lanes."""
    g = GROUPS[groups]
    c = S.Batch(g, _own(g, own, 5), hq, hkv, hd, dt, seed=7, page=32, int8=int8)
    c.run()
    c.check(c.out)


@pytest.mark.parametrize("page", [16, 128, 1024])
def test_pages(page):
    g = [(4, 3 * page + 5), (3, page), (2, page - 1), (1, 2 * page + 1)]
    c = S.Batch(g, [0, 1, page, page + 1, 17, 2 * page, 5, 3, 64, 31], 8, 2, 128, BF, seed=11, page=page)
    c.run()
    c.check(c.out)


def test_is_decode_over_repeated_tables():
    """The same as attn_decode over tables that name the prefix's pages in front of each sequence's."""
    from qwen35_amd.kernels import attention as A
    page, pre = 64, 6 * 64
    own = [1, 30, 64, 65, 200, 7]
    c = S.Batch([(6, pre)], own, 8, 2, 256, BF, seed=13, page=page)
    c.run()
    k, v, _, _ = c.cache
    table = torch.cat([c.ptable[:, :pre // page].expand(6, -1), c.table], 1).contiguous()
    lens = torch.tensor([pre + n for n in own], dtype=torch.int32, device="cuda")
    y = A.attn_decode(c.q, k, v, table, lens, torch.empty_like(c.q))
    ref, tol = c.expected()
    R.check(y, ref, tol)
    R.check(c.out, ref, tol)


def test_views_and_strides():
    """Queries as part of a projection's rows, output rows with room between them, a table with wide rows,
    lengths in front of larger tensors."""
    c = S.Batch([(3, 100), (2, 65)], [5, 0, 33, 64, 1], 8, 2, 64, F16, seed=17, page=16)
    proj = torch.zeros((5, 8, 2 * 64), dtype=F16, device="cuda")
    proj[..., :64] = c.q
    room = torch.full((5, 8, 3 * 64), 5.0, dtype=F16, device="cuda")
    wide = torch.full((5, c.table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    c.run(q=proj[..., :64], out=room[..., 64:128], table=wide[:, :c.table.shape[1]])
    c.check(room[..., 64:128])
    assert bool((room[..., :64] == 5).all()) and bool((room[..., 128:] == 5).all())


def test_same_bits_again():
    c = S.Batch([(8, 5000), (3, 77)], [9 * i for i in range(11)], 8, 2, 256, BF, seed=19)
    first = c.run().clone()
    for _ in range(5):
        assert torch.equal(c.run(), first)


def test_groups_do_not_see_each_other():
    """A group's keys of no number, and own keys of another sequence, reach nobody else; keys behind the
    lengths neither."""
    c = S.Batch([(2, 40), (2, 50)], [3, 17, 20, 31], 4, 1, 128, BF, seed=23, page=16)
    k, v, _, _ = c.cache
    ref, tol = c.expected()
    k[c.ptable[0, 0].long()] = float("nan")
    v[c.table[2, 0].long()] = float("inf")
    # places behind the ends of prefix 1 (2 of its last page) and of sequence 1 (1 of its second)
    k[c.ptable[1, 3].long(), 2:] = float("nan")
    v[c.ptable[1, 3].long(), 2:] = float("inf")
    v[c.table[1, 1].long(), 1:] = float("nan")
    c.run()
    assert bool(c.out[:2].isnan().all())
    assert not bool(c.out[2].isfinite().any())
    R.check(c.out[3:], ref[3:], tol[3:])


def test_bad_pages_lengths_and_bounds():
    """What the device finds in tables, lengths and bounds has a stated result, and touches no memory
    outside the cache."""
    c = S.Batch([(2, 40), (2, 50), (1, 20)], [3, 17, 20, 31, 8], 4, 1, 128, BF, seed=29, page=16)
    ref, tol = c.expected()
    # a page outside the cache in the middle group's prefix, and behind the first one's end
    c.ptable[1, 1] = 1 << 30
    c.ptable[0, 3] = -5
    c.run()
    assert bool(c.out[2:4].isnan().all())
    R.check(c.out[[0, 1, 4]], ref[[0, 1, 4]], tol[[0, 1, 4]])
    # one in a sequence's own pages
    c = S.Batch([(2, 40), (2, 50), (1, 20)], [3, 17, 20, 31, 8], 4, 1, 128, BF, seed=29, page=16)
    c.table[3, 0] = -1
    c.run()
    assert bool(c.out[3].isnan().all())
    R.check(c.out[[0, 1, 2, 4]], ref[[0, 1, 2, 4]], tol[[0, 1, 2, 4]])
    # lengths below zero are none; those past a table what it holds
    c = S.Batch([(2, 40), (2, 64), (1, 0)], [3, 17, 48, 31, 0], 4, 1, 128, BF, seed=31, page=16)
    ref, tol = c.expected()
    c.plen[2], c.len[4] = -7, -(1 << 31)
    c.plen[1], c.len[2] = 1 << 30, (1 << 31) - 1
    c.run(prefix_table=c.ptable[:, :4], table=c.table[:, :3])
    R.check(c.out, ref, tol)
    # bounds that fall, and those outside the batch
    c = S.Batch([(2, 40), (0, 64), (3, 20)], [3, 17, 48, 31, 0], 4, 1, 128, BF, seed=37, page=16, pad=2)
    ref, tol = c.expected()
    c.cu.copy_(torch.tensor([0, 2, 1, 5], dtype=torch.int32))
    c.run()
    R.check(c.out[:5], ref, tol)
    assert bool((c.out[5:] == 7).all())
    c.out.fill_(7.0)
    c.cu.copy_(torch.tensor([-9, 2, -1, 1 << 30], dtype=torch.int32))
    c.run()
    R.check(c.out[:5], ref, tol)


def test_empty_calls_and_tables():
    from qwen35_amd.kernels import attention as A
    c = S.Batch([(2, 40)], [0, 0], 4, 1, 64, BF, seed=41, page=16)
    c.run(table=c.table[:, :0])
    c.check(c.out)
    c.run(table=c.table[:, :0], prefix_table=c.ptable[:, :0])
    assert bool((c.out == 0).all())
    c.out.fill_(7.0)
    c.run(prefix_table=c.ptable[:0], prefix_len=c.plen[:0], cu_seq=c.cu[:1])   # no groups
    assert bool((c.out == 7).all())
    k, v, _, _ = c.cache
    A.attn_decode_shared(c.q[:0], k, v, c.ptable, c.plen, c.cu, c.table[:0], c.len[:0], c.out[:0])


@pytest.mark.parametrize("hq,hd,int8", [(8, 256, False), (16, 128, True)])
def test_graph_replays_with_other_lengths(hq, hd, int8):
    from qwen35_amd.kernels import qlin as C
    c = S.Batch([(4, 600), (3, 100)], [64, 3, 10, 0, 50, 20, 33], hq, 2, hd, BF, seed=43, page=16, int8=int8)
    c.run()
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        c.run()
    for plen, lens, cu in (([600, 100], [64, 3, 10, 0, 50, 20, 33], [0, 4, 7]), ([1, 77], [1] * 7, [0, 1, 7]),
                           ([300, 0], [0, 0, 9, 8, 7, 6, 5], [0, 7, 7]), ([600, 100], [64, 3, 10, 0, 50, 20, 33], [0, 4, 6])):
        for t, x in ((c.plen, plen), (c.len, lens), (c.cu, cu)):
            t.copy_(torch.tensor(x, dtype=torch.int32))
        c.groups, c.own = [(cu[1] - cu[0], plen[0]), (cu[2] - cu[1], plen[1])], lens
        eager = c.run(out=torch.full_like(c.out, 7.0)).clone()
        c.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out.view(torch.int16), eager.view(torch.int16))
        # (the fourth sequence has no page of its own: one that it names lies outside the cache)
        ref, tol = c.expected()
        some = [b for b in range(cu[2]) if b != 3 or lens[3] == 0]
        R.check(c.out[some], ref[some], tol[some])
        assert bool(c.out[3].isnan().all()) == (lens[3] > 0)
        assert bool((c.out[cu[2]:] == 7).all())


def test_two_streams():
    from qwen35_amd.kernels import qlin as C
    cs = [S.Batch([(8, 3000 + 100 * i)], [7 * j for j in range(8)], 8, 2, 128, BF, seed=47 + i) for i in range(2)]
    want = [c.run().clone() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    for s in streams:
        C.bind_workspace(s)
    torch.cuda.synchronize()
    outs = [[] for _ in cs]
    for _ in range(4):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                outs[i].append(c.run(out=torch.empty_like(c.out)))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for o in outs[i]:
            assert torch.equal(o, w)


def test_light_keys_beside_a_heavy_one():
    """fp16: keys 24 octaves lighter than one of the prefix's keep their weight, whichever part they
    are in (their sum decides a column)."""
    page, hd = 64, 64
    c = S.Batch([(2, 4096)], [4096, 100], 1, 1, hd, F16, seed=53, page=page, scale=1.0)
    k, v, _, _ = c.cache
    k.zero_(), v.zero_()
    c.q.zero_()
    c.q[:, :, 0] = 1.0
    k[c.ptable[0, 0].long(), 0, 0, 0] = 17.0                 # 24.5 octaves above the others
    for t, n in ((c.ptable[0], 4096), (c.table[0], 4096), (c.table[1], 100)):
        v[t[:-(-n // page)].long(), :, 0, 1] = 30000.0
    v[c.ptable[0, 0].long(), 0, 0, 1] = 0.0
    c.run()
    c.check(c.out)


def test_large_scores_and_offsets():
    """Scores of a large deviation, and parts whose references lie far from each other."""
    for dt in (BF, F16):
        c = S.Batch([(4, 900)], [100, 1, 33, 64], 8, 2, 128, dt, seed=59, page=16, scale=1.0)
        k, _, _, _ = c.cache
        k[c.ptable[0, :20].long()] *= 3
        c.run()
        c.check(c.out)


def test_many_sequences():
    """A thousand sequences in groups of all sizes; and more than the workspace holds sums of are refused."""
    rng = random.Random(61)
    groups = []
    while sum(n for n, _ in groups) < 1000:
        groups.append((rng.choice([0, 1, 2, 5, 30, 90]), rng.choice([0, 1, 20, 200])))
    c = S.Batch(groups, _own(groups, 30, 67), 4, 2, 64, BF, seed=71, page=16)
    c.run()
    c.check(c.out)
    k, v, _, _ = c.cache
    from qwen35_amd.kernels import attention as A
    n = 1 << 16
    q = torch.empty((n, 8, 64), dtype=BF, device="cuda")
    table = torch.zeros((n, 1), dtype=torch.int32, device="cuda")
    one = torch.ones(n, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="more than the workspace holds"):
        A.attn_decode_shared(q, k, v, c.ptable, c.plen, c.cu, table, one, torch.empty_like(q))


def test_cache_past_4_gib():
    """Pages whose byte offsets pass 32 bits, in the prefix and in a sequence's own keys."""
    hd, hkv, page = 128, 2, 64
    pages = 70000                                            # 70000 x 64 x 2 x 128 x 2 bytes: 2.3 GB each
    k = torch.zeros((pages, page, hkv, hd), dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    c = S.Batch([(4, 300)], [70, 5, 64, 1], 8, hkv, hd, BF, seed=73, page=page)
    far = lambda t: torch.where(t >= 0, pages - 1 - t * 7, t)
    for t in (c.ptable, c.table):
        ids = t[t >= 0].long()
        k[far(ids)], v[far(ids)] = c.cache[0][ids], c.cache[1][ids]
    ref, tol = c.expected()
    c.cache = (k, v, None, None)
    c.run(prefix_table=far(c.ptable), table=far(c.table))
    R.check(c.out, ref, tol)


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [3, 20])
def test_odd_queries(dt, int8, n):
    """A query that is no number, infinite, zero or tiny concerns its own head of its own sequence alone."""
    c = S.Batch([(n, 300)], [40 + i for i in range(n)], 8, 2, 128, dt, seed=79, int8=int8, page=16)
    c.q[0, 3, 7] = float("nan")
    c.q[1, 5, 0] = float("inf")
    c.q[2, 0] = 0.0
    c.q[2, 1] *= 2.0 ** -14
    c.run()
    ref, tol = c.expected()
    odd = torch.zeros((n, 8), dtype=torch.bool, device="cuda")
    odd[0, 3] = odd[1, 5] = True
    assert bool(c.out[odd].isnan().all())
    R.check(c.out[~odd], ref[~odd], tol[~odd])


@pytest.mark.parametrize("hq,hkv", [(8, 2), (32, 1)])
def test_odd_scales(hq, hkv):
    """An int8 cache's scales that are not finite: a key's makes no number of what sees it, whatever its score's
    sign, and places behind the end may hold anything."""
    c = S.Batch([(4, 100), (3, 40)], [5, 20, 33, 1, 7, 0, 9], hq, hkv, 128, BF, seed=83, page=16, int8=True)
    _, _, ks, vs = c.cache
    ref, tol = c.expected()
    ks[c.ptable[0, 6].long(), 4:] = float("inf")      # behind the first prefix's end
    vs[c.table[1, 1].long(), 4:] = float("nan")       # behind the second sequence's
    ks[c.table[4, 0].long(), 3] = float("-inf")       # a key of the fifth sequence
    c.run()
    some = [0, 1, 2, 3, 5, 6]
    R.check(c.out[some], ref[some], tol[some])
    assert bool(c.out[4].isnan().all())


def test_infinite_values_behind_the_end():
    """Wide tiles zero the values behind the last key, which hold it again: an infinite last value stays in its own
    column (and makes that column infinite)."""
    for n in (2, 40):
        c = S.Batch([(n, 77)], [0] * n, 4, 1, 128, BF, seed=89, page=16)
        _, v, _, _ = c.cache
        v[c.ptable[0, 4].long(), 12, 0, 5] = float("inf")     # the 77th key's
        ref, tol = c.expected()
        c.run()
        assert bool((c.out[..., 5] == float("inf")).all())
        rest = [i for i in range(128) if i != 5]
        v[c.ptable[0, 4].long(), 12, 0, 5] = 0.0
        ref, tol = c.expected()
        R.check(c.out[..., rest], ref[..., rest], tol[..., rest])
