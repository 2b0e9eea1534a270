"""attn_prompt and attn_prompt_paged against attention in 64 bits."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _packed(nq, hq, hkv, hd, dt, nk=None, causal=True, seed=0, scale=None, spoil=None, tail=0):
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, Tk = sum(nq) + tail, sum(nk or nq) + tail
    q = torch.randn((T, hq, hd), generator=g, device="cuda").to(dt) * 2
    kv = torch.randn((Tk, 2 * hkv * hd), generator=g, device="cuda").to(dt)
    k, v = kv[:, :hkv * hd].view(Tk, hkv, hd), kv[:, hkv * hd:].view(Tk, hkv, hd)
    if tail:
        kv[Tk - tail:] = torch.nan
    if spoil:
        spoil(q, k, v)
    out = torch.full((T, hq, hd), 7.0, dtype=dt, device="cuda")
    A.attn_prompt(q, k, v, _cu(nq), out, cu_k=_cu(nk) if nk else None, scale=scale, causal=causal)
    torch.cuda.synchronize()
    at = ak = 0
    for b, (m, n) in enumerate(zip(nq, nk or nq)):
        seen = R.causal(m, n, "cuda") if causal else torch.ones((m, n), dtype=torch.bool, device="cuda")
        if not spoil:
            ref, tol = R.attend(q[at:at + m], k[ak:ak + n], v[ak:ak + n], scale or hd ** -0.5, seen, dt)
            R.check(out[at:at + m], ref, tol, f"sequence {b} ({m}, {n})")
        at, ak = at + m, ak + n
    if tail:
        assert (out[T - tail:] == 7).all()
    return out, q, k, v


def _paged(nq, past, hq, hkv, hd, dt, page=64, int8=False, causal=True, seed=0, head_major=True):
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = [a + b for a, b in zip(nq, past)]
    table, pages = R.pages_of(lens, page, 3, seed, "cuda")
    c = R.cache(pages, page, hkv, hd, dt, seed + 1, int8, head_major)
    if not int8:
        own = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                own[table[b, i].long(), :min(page, n - i * page)] = True
        for x in c[:2]:
            x[~own] = torch.nan
    T = sum(nq)
    q = torch.randn((T, hq, hd), generator=g, device="cuda").to(dt) * 2
    out = torch.full((T, hq, hd), 7.0, dtype=dt, device="cuda")
    A.attn_prompt_paged(q, c[0], c[1], table, torch.tensor(lens, dtype=torch.int32, device="cuda"), _cu(nq), out,
                        k_s=c[2], v_s=c[3], causal=causal)
    torch.cuda.synchronize()
    at = 0
    for b, (m, n) in enumerate(zip(nq, lens)):
        k, v = R.gathered(c, table, b, n)
        seen = R.causal(m, n, "cuda") if causal else torch.ones((m, n), dtype=torch.bool, device="cuda")
        ref, tol = R.attend(q[at:at + m], k, v, hd ** -0.5, seen, dt, 2.0 ** -16 if int8 and dt == FP else None)
        R.check(out[at:at + m], ref, tol, f"sequence {b} ({m}, {n})")
        at += m
    return out


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 200, 513])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_one_prompt(n, hd, causal):
    _packed([n], 8, 2, hd, BF, causal=causal, seed=n)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (20, 5), (40, 2), (64, 1), (16, 8)])
@pytest.mark.parametrize("dt", [BF, FP])
def test_head_groups(hq, hkv, dt):
    _packed([150, 0, 1, 77], hq, hkv, 128, dt, seed=hq)
    _packed([130], hq, hkv, 256, dt, seed=hq)


def test_packed_prompts_with_rows_behind_them():
    _packed([5, 0, 300, 64, 1, 0, 129], 8, 2, 256, BF, seed=1, tail=37)
    _packed([(i * 31) % 97 for i in range(100)], 4, 4, 64, FP, seed=2, tail=1)


def test_other_numbers_of_keys():
    """Fewer keys than queries leave the first rows empty; more are a past."""
    _packed([40, 100, 3, 9, 0, 33], 8, 2, 256, BF, nk=[17, 400, 0, 9, 5, 1], seed=3)
    _packed([40, 100, 3, 9, 0, 33], 8, 2, 128, FP, nk=[17, 400, 0, 9, 5, 1], seed=3, causal=False)


def test_long_prompt_is_cut_and_joined():
    _packed([3333], 8, 2, 256, BF, seed=4)
    _packed([2050, 90], 4, 1, 128, FP, seed=5)
    _packed([1500], 2, 1, 64, BF, seed=6)


def test_many_tiles_are_cut_and_joined_by_their_last_part():
    _packed([4200, 0, 1700, 33], 8, 2, 256, BF, seed=15, tail=5)
    _packed([5000, 700], 16, 2, 64, FP, seed=16)
    _packed([17] * 70 + [4500], 8, 2, 128, BF, seed=17)


def test_ragged_batches_in_one_piece():
    _packed([900, 3, 0, 899, 450, 64, 1, 700], 8, 2, 256, BF, seed=18, tail=3)
    _packed([(i * 37) % 400 for i in range(64)], 16, 4, 64, FP, seed=19)
    _packed([(i * 37) % 400 for i in range(65)], 16, 4, 64, FP, seed=19, causal=False)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,dt", [(64, BF), (128, FP), (256, BF), (256, FP)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_chunks_over_the_cache(int8, hd, dt, page):
    _paged([100, 1, 33], [513, 0, 77], 8, 2, hd, dt, page=page, int8=int8, seed=page + hd, head_major=page != 64)


@pytest.mark.parametrize("int8", [False, True])
def test_long_chunks_over_the_cache(int8):
    _paged([512], [6000], 8, 2, 256, BF, int8=int8, seed=7)
    _paged([7], [20000], 8, 2, 128, FP, page=16, int8=int8, seed=8)
    _paged([65, 3], [100, 3000], 3, 3, 64, BF, page=32, int8=int8, seed=9, causal=False)


def test_a_masked_key_has_no_part_whatever_it_holds():
    """Values that are no numbers in the last third of the prompt: the rows in front of them are
    what they are without, the first row that sees one is not."""
    for nq, hd, dt in (([90], 256, BF), ([700], 256, BF), ([90], 64, FP), ([1200], 128, FP)):
        bad = 2 * nq[0] // 3

        def spoil(q, k, v):
            v[bad, 0, 3] = torch.nan
            v[bad + 2, 1, 5] = torch.inf
            k[bad + 1, :, 0] = torch.nan

        out, q, k, v = _packed(nq, 8, 2, hd, dt, seed=11, spoil=spoil)
        ref, tol = R.attend(q[:bad], k[:bad], v[:bad], hd ** -0.5, R.causal(bad, bad, "cuda"), dt)
        R.check(out[:bad], ref, tol, "rows in front")
        assert out[bad:, :4, 3].isnan().all()
        assert out[bad + 1:].isnan().all()
        assert out[bad, 4:].isfinite().all()


@pytest.mark.parametrize("nq,nk", [(1, 1), (3, 37), (90, 90), (40, 3000)])
def test_an_infinite_value_is_of_its_own_column(nq, nk):
    """The last key's place is taken again behind it: its infinity must not meet a weight of zero
    there."""
    def spoil(q, k, v):
        v[-1, 1, 77] = torch.inf

    out, q, k, v = _packed([nq], 8, 2, 128, BF, nk=[nk], seed=14, spoil=spoil, causal=False)
    assert (out[:, 4:, 77] == torch.inf).all()
    seen = torch.ones((nq, nk), dtype=torch.bool, device="cuda")
    ref, tol = R.attend(q, k, v, 128 ** -0.5, seen, BF)
    rest = torch.ones_like(ref, dtype=torch.bool)
    rest[:, 4:, 77] = False
    R.check(out[rest], ref[rest], tol[rest])


def test_a_score_of_minus_infinity_is_no_weight():
    def spoil(q, k, v):
        k[:40, :, 0] = -torch.inf
        q[..., 0] = 1.0

    out, q, k, v = _packed([100], 8, 2, 128, BF, seed=13, spoil=spoil)
    assert out[:40].isnan().all()                    # nothing but -inf: 0 / 0
    seen = R.causal(100, 100, "cuda")
    seen[:, :40] = False
    ref, tol = R.attend(q, k.nan_to_num(0, 0, 0), v, 128 ** -0.5, seen, BF)
    R.check(out[40:], ref[40:], tol[40:])


def test_repeats_are_the_same_bits():
    a = _packed([2100, 77], 8, 2, 256, BF, seed=12)[0]
    for _ in range(4):
        assert torch.equal(a, _packed([2100, 77], 8, 2, 256, BF, seed=12)[0])


def test_nothing_to_do():
    from qwen35_amd.kernels import attention as A
    e = torch.empty((0, 2, 64), dtype=BF, device="cuda")
    A.attn_prompt(e, e, e, _cu([0]), e)
    q = torch.full((3, 2, 64), 5.0, dtype=BF, device="cuda")
    out = torch.full_like(q, 7.0)
    A.attn_prompt(q, e, e, _cu([3]), out, cu_k=_cu([0]))      # queries without a key
    assert (out == 0).all()
    A.attn_prompt(q, q, q, _cu([]), out)                        # no sequence: rows stay
    assert (out == 0).all()
