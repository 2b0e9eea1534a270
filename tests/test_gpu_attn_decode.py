"""attn_decode against attention in 64 bits."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _run(lens, hq, hkv, hd, dt, page=64, int8=False, seed=0, head_major=True, scale=None, spoil=True):
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(seed)
    table, pages = R.pages_of(lens, page, 3, seed, "cuda")
    c = R.cache(pages, page, hkv, hd, dt, seed + 1, int8, head_major)
    if spoil and not int8:
        # what lies behind a sequence's last key is nobody's: numbers must not be needed there
        own = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                own[table[b, i].long(), :min(page, n - i * page)] = True
        for x in c[:2]:
            x[~own] = torch.nan
    q = torch.randn((len(lens), hq, hd), generator=g, device="cuda").to(dt) * 2
    out = torch.full((len(lens), hq, hd), 7.0, dtype=dt, device="cuda")
    kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    A.attn_decode(q, c[0], c[1], table, kv_len, out, k_s=c[2], v_s=c[3], scale=scale)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        k, v = R.gathered(c, table, b, n)
        seen = torch.ones((1, n), dtype=torch.bool, device="cuda")
        ref, tol = R.attend(q[b:b + 1], k, v, scale or hd ** -0.5, seen, dt, 2.0 ** -16 if int8 else None)
        R.check(out[b:b + 1], ref, tol, f"sequence {b} of {n} keys")
    return out


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 1000, 4097])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("int8", [False, True])
def test_one_sequence(n, hd, int8):
    _run([n], 8, 2, hd, BF, int8=int8, seed=n + hd)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (20, 5), (16, 1), (17, 1), (40, 2), (64, 1)])
@pytest.mark.parametrize("int8", [False, True])
def test_head_groups(dt, hq, hkv, int8):
    _run([300, 0, 77, 640], hq, hkv, 128, dt, page=16, int8=int8, seed=hq)
    _run([513], hq, hkv, 256, dt, page=32, int8=int8, seed=hq + 1)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("head_major", [False, True])
def test_pages_and_layouts(page, head_major):
    _run([1, 0, 2047, 16, 1025], 8, 2, 256, BF, page=page, head_major=head_major, seed=page)
    _run([1, 0, 2047, 16, 1025], 8, 2, 64, FP, page=page, head_major=head_major, seed=page, int8=True)


def test_ragged_batches_of_more_than_a_wave():
    lens = [(37 * i * i) % 700 for i in range(150)]
    _run(lens, 4, 2, 128, BF, page=16, seed=5)


def test_long_contexts_join_in_two_steps():
    _run([70001], 8, 2, 256, BF, seed=8, spoil=False)
    _run([131072 + 5, 3], 4, 1, 128, FP, page=128, int8=True, seed=9)


def test_peaked_scores_and_scale():
    _run([900], 8, 2, 256, BF, seed=3, scale=1.5)
    _run([900], 8, 2, 256, FP, seed=4, scale=1e-3)


def test_repeats_are_the_same_bits():
    a = _run([9001, 40, 0, 3000], 8, 2, 256, BF, seed=12)
    for _ in range(5):
        assert torch.equal(a, _run([9001, 40, 0, 3000], 8, 2, 256, BF, seed=12))


@pytest.mark.parametrize("n", [1, 37, 5000])
@pytest.mark.parametrize("int8", [False, True])
def test_an_infinite_value_is_of_its_own_column(n, int8):
    """The last key's place is taken again behind it: its infinity must not meet a weight of zero
    there."""
    from qwen35_amd.kernels import attention as A
    table, pages = R.pages_of([n], 64, 2, n, "cuda")
    c = R.cache(pages, 64, 2, 128, BF, n + 1, int8)
    last = (int(table[0, (n - 1) // 64]), (n - 1) % 64)
    rest = torch.ones((2, 128), dtype=torch.bool, device="cuda")
    if int8:
        c[3][last][0] = torch.inf
        rest[0] = False
    else:
        c[1][last][1, 77] = torch.inf
        rest[1, 77] = False
    q = torch.randn((1, 8, 128), device="cuda").to(BF)
    out = torch.empty_like(q)
    kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
    A.attn_decode(q, c[0], c[1], table, kv_len, out, k_s=c[2], v_s=c[3])
    k, v = R.gathered(c, table, 0, n)
    rest = rest.repeat_interleave(4, 0)[None]
    if int8:
        assert not out[~rest].isfinite().any()
    else:
        assert (out[~rest] == torch.inf).all()
    seen = torch.ones((1, n), dtype=torch.bool, device="cuda")
    ref, tol = R.attend(q, k, v, 128 ** -0.5, seen, BF, 2.0 ** -16 if int8 else None)
    R.check(out[rest], ref[rest], tol[rest])
