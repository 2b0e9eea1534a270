"""Caches at the ends of what the calls accept: heads further apart than a token's stride may be, [kv_heads,
pages, page, hd], written by qk_norm_rope, read by a chunk and by a decode step; a table of no pages."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("int8", [False, True])
def test_heads_of_more_than_a_token_stride(int8):
    from qwen35_amd.kernels import attention as A
    page, hkv, hd, hq = 64, 2, 64, 8
    pages = (1 << 26) // (page * hd) + 9
    dt = torch.int8 if int8 else BF
    kc, vc = (torch.zeros((hkv, pages, page, hd), dtype=dt, device="cuda").permute(1, 2, 0, 3) for _ in range(2))
    ks, vs = ((torch.zeros((hkv, pages, page), device="cuda").permute(1, 2, 0) for _ in range(2)) if int8
              else (None, None))
    assert kc.stride(2) > 1 << 26
    n, g = 700, torch.Generator("cuda").manual_seed(1)
    table = torch.randperm(pages, generator=g, device="cuda")[:-(-n // page)].to(torch.int32)[None]
    x = torch.randn((n, (hq + 2 * hkv) * hd), generator=g, device="cuda").to(BF)
    q, k, v = (t.view(n, -1, hd) for t in x.split([hq * hd, hkv * hd, hkv * hd], 1))
    i = torch.arange(n, device="cuda")
    slots = table[0].long()[i // page] * page + i % page
    freqs = torch.tensor([1e4 ** (-j / 32) for j in range(32)], dtype=torch.float64, device="cuda")
    qr = torch.empty((n, hq, hd), dtype=BF, device="cuda")
    A.qk_norm_rope(q, k, i, freqs, qr, v=v, k_cache=kc, v_cache=vc, slots=slots, k_s=ks, v_s=vs)
    kk, vv = R.gathered((kc, vc, ks, vs), table, 0, n)
    assert int8 or torch.equal(vv.to(BF), v)
    assert (vv - v.double()).abs().max() <= (v.abs().max() / 127 if int8 else 0)
    out, one = torch.empty_like(qr), torch.empty_like(qr[:1])
    kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
    A.attn_prompt_paged(qr, kc, vc, table, kv_len, torch.tensor([0, n], dtype=torch.int32, device="cuda"), out, k_s=ks,
                        v_s=vs)
    A.attn_decode(qr[-1:], kc, vc, table, kv_len, one, k_s=ks, v_s=vs)
    ref, tol = R.attend(qr, kk, vv, hd ** -0.5, R.causal(n, n, "cuda"), BF)
    R.check(out, ref, tol, "prompt")
    R.check(one, ref[-1:], tol[-1:], "decode")


def test_a_table_of_no_pages_gives_zeros():
    from qwen35_amd.kernels import attention as A
    c = R.cache(4, 16, 2, 64, BF, 1)
    table = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([0, 5, 0], dtype=torch.int32, device="cuda")
    q = torch.randn((3, 8, 64), device="cuda").to(BF)
    for call in (lambda o: A.attn_decode(q, c[0], c[1], table, kv_len, o),
                 lambda o: A.attn_prompt_paged(q, c[0], c[1], table, kv_len,
                                               torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"), o)):
        out = torch.full_like(q, 7)
        call(out)
        assert (out == 0).all()
