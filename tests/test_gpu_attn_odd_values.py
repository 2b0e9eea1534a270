"""Infinities and NaN among the values of a prompt, before and behind a row's last key: a row's output is
what the values that it sees add up to, and what it does not see has no part in it -- at the cost of a
second pass over the keys."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
INF, NAN = torch.inf, torch.nan


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check(out, q, k, v, seen, dt, name):
    """`k` finite, `v` [n, hkv, hd] with anything in it."""
    hq, hkv = q.shape[1], k.shape[1]
    ref, tol = R.attend(q, k, v, q.shape[-1] ** -0.5, seen, dt)
    for h in range(hq):
        x = v[:, h // (hq // hkv)].float()
        plus, minus, nan = ((seen.float() @ m.float()) > 0 for m in (x == INF, x == -INF, x.isnan()))
        y = out[:, h].double()
        none = nan | (plus & minus)
        assert y[none].isnan().all(), name
        assert (y[plus & ~none] == INF).all() and (y[minus & ~none] == -INF).all(), name
        rest = ~(plus | minus | nan)
        R.check(y[rest], ref[:, h][rest], tol[:, h][rest], f"{name}, head {h}")


def _sprinkle(v, g, many):
    """Odd values in `many` places of v [n, hkv, hd], in few columns, so that others stay numbers."""
    n, hkv, hd = v.shape
    at = torch.randint(0, n, (many,), generator=g)
    at[:3] = torch.tensor([0, n - 1, n // 2])
    cols = torch.randint(0, hd, (many,), generator=g) // 4 * 4
    for i, (j, c) in enumerate(zip(at.tolist(), cols.tolist())):
        v[j, i % hkv, c] = (INF, -INF, NAN, INF)[i % 4]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("nq,nk,causal", [(1, 1, True), (40, 40, True), (33, 33, False), (64, 1500, True), (700, 700, True),
                                          (900, 500, True), (2600, 2600, True), (130, 1001, False)])
def test_packed(hd, dt, nq, nk, causal):
    """Halved and whole tiles, cut and uncut, joined either way."""
    from qwen35_amd.kernels import attention as A
    g = torch.Generator().manual_seed(nq + nk + hd)
    hq, hkv = (8, 2) if nq < 2000 else (4, 2)
    q, k, v = (torch.randn((n, h, hd), generator=g).to(dt).cuda() for n, h in ((nq, hq), (nk, hkv), (nk, hkv)))
    _sprinkle(v, g, 6 + nk // 60)
    out = torch.empty_like(q)
    A.attn_prompt(q, k, v, _ints(0, nq), out, cu_k=_ints(0, nk), causal=causal)
    seen = R.causal(nq, nk, "cuda") if causal else torch.ones((nq, nk), dtype=torch.bool, device="cuda")
    _check(out, q, k, v, seen, dt, f"{nq} over {nk}")


def test_many_whole_tiles_of_a_batch():
    from qwen35_amd.kernels import attention as A
    g = torch.Generator().manual_seed(3)
    lens, hd = [700, 0, 450, 33, 900, 64, 650, 800], 256
    T = sum(lens)
    q, k, v = (torch.randn((T, h, hd), generator=g).to(BF).cuda() for h in (8, 2, 2))
    cu, at = [0], 0
    for b, n in enumerate(lens):
        if n and b % 2 == 0:
            _sprinkle(v[at:at + n], g, 9)
        at += n
        cu.append(at)
    out = torch.empty_like(q)
    A.attn_prompt(q, k, v, _ints(*cu), out)
    for b, n in enumerate(lens):
        s = slice(cu[b], cu[b + 1])
        if n:
            _check(out[s], q[s], k[s], v[s], R.causal(n, n, "cuda"), BF, f"prompt {b}")


@pytest.mark.parametrize("nq,past", [([70, 5], [0, 900]), ([512], [4000]), ([3], [9000])])
def test_over_the_cache(nq, past):
    from qwen35_amd.kernels import attention as A
    g = torch.Generator().manual_seed(sum(past))
    hd, page = 128, 32
    lens = [a + b for a, b in zip(nq, past)]
    table, pages = R.pages_of(lens, page, 1, 4, "cuda")
    kc, vc = R.cache(pages, page, 2, hd, BF, 5)[:2]
    q = torch.randn((sum(nq), 8, hd), generator=g).to(BF).cuda()
    out = torch.empty_like(q)
    for b, n in enumerate(lens):
        v = torch.zeros((n, 2, hd), dtype=BF, device="cuda")
        _sprinkle(v, g, 12)
        i = torch.arange(n, device="cuda")
        p, o = table[b].long()[i // page], i % page
        vc[p, o] = torch.where(v == 0, vc[p, o], v)
    A.attn_prompt_paged(q, kc, vc, table, _ints(*lens), _ints(0, *torch.tensor(nq).cumsum(0).tolist()), out)
    at = 0
    for b, (m, n) in enumerate(zip(nq, lens)):
        i = torch.arange(n, device="cuda")
        p, o = table[b].long()[i // page], i % page
        _check(out[at:at + m], q[at:at + m], kc[p, o], vc[p, o], R.causal(m, n, "cuda"), BF, f"sequence {b}")
        at += m


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,past", [(60, 0), (400, 300), (9, 5000)])
def test_scales_that_are_no_numbers(dt, hd, nq, past):
    """An int8 cache: a key whose key or value scale is not finite makes no number of every row of its
    head that sees it, and of no other."""
    from qwen35_amd.kernels import attention as A
    n, page = nq + past, 64
    table, pages = R.pages_of([n], page, 1, 4, "cuda")
    c = R.cache(pages, page, 2, hd, dt, 6, True)
    ok = [x.clone() for x in R.gathered(c, table, 0, n)]
    q = torch.randn((nq, 8, hd), generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(dt)
    first = n - nq + nq // 3
    for i, (x, bad) in enumerate(((c[2], INF), (c[3], NAN), (c[2], -INF), (c[3], INF), (c[3], -INF), (c[2], NAN))):
        j = min(first + 3 * i, n - 1)
        x[table[0, j // page].long(), j % page, 0] = bad
        if i == 0:
            other = min(j + 5, n - 1)
            c[3][table[0, other // page].long(), other % page, 1] = NAN
    out = torch.empty_like(q)
    A.attn_prompt_paged(q, c[0], c[1], table, _ints(n), _ints(0, nq), out, k_s=c[2], v_s=c[3])
    seen = R.causal(nq, n, "cuda")
    ref, tol = R.attend(q, *ok, hd ** -0.5, seen, dt, None if dt == BF else 2.0 ** -16)
    for head, at in ((0, first), (1, other)):
        sees = seen[:, at]
        h = slice(4 * head, 4 * head + 4)
        assert out[sees][:, h].isnan().all(), (head, at)
        R.check(out[~sees][:, h], ref[~sees][:, h], tol[~sees][:, h], f"key head {head}")


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("n,at", [(1, 0), (45, 44), (3000, 1234), (70000, 69000)])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("of_values", [False, True])
def test_a_decode_step_over_a_scale_that_is_no_number(hd, n, at, bad, of_values):
    """Whatever the sign of its scores; the other key head is what it is."""
    from qwen35_amd.kernels import attention as A
    table, pages = R.pages_of([n], 64, 1, 4, "cuda")
    c = R.cache(pages, 64, 2, hd, BF, 7, True)
    ok = [x.clone() for x in R.gathered(c, table, 0, n)]
    q = torch.randn((1, 32, hd), generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(BF)
    c[3 if of_values else 2][table[0, at // 64].long(), at % 64, 1] = bad
    out = torch.empty_like(q)
    A.attn_decode(q, c[0], c[1], table, _ints(n), out, k_s=c[2], v_s=c[3])
    assert out[:, 16:].isnan().all()
    ref, tol = R.attend(q, *ok, hd ** -0.5, torch.ones((1, n), dtype=torch.bool, device="cuda"), BF, 2.0 ** -16)
    R.check(out[:, :16], ref[:, :16], tol[:, :16])


def test_one_value_costs_no_more_than_another_pass():
    """A NaN in the first key's value, which every row sees: about three times the time, not hundreds."""
    from qwen35_amd.kernels import attention as A
    T, hd = 4096, 256
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v = (torch.randn((T, h, hd), generator=g, device="cuda").to(BF) for h in (8, 2, 2))
    out, cu = torch.empty_like(q), _ints(0, T)
    best = []
    for bad in (False, True):
        if bad:
            v[0, :, 7] = NAN
        A.attn_prompt(q, k, v, cu, out)
        times = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            A.attn_prompt(q, k, v, cu, out)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        best.append(min(times))
    assert best[1] < 12 * best[0], best
    rest = torch.arange(hd, device="cuda") != 7
    assert out[..., 7].isnan().all() and out[..., rest].isfinite().all()
