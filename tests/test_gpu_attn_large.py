"""The attention operators' largest calls: very many sequences, very long ones (single rows of the
output against attention in 64 bits)."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _rows(out, q, k, v, rows, seen_of, dt, name, up=None):
    hd = q.shape[-1]
    for i in rows:
        n = seen_of(i)
        seen = torch.ones((1, n), dtype=torch.bool, device="cuda")
        ref, tol = R.attend(q[i:i + 1], k[:n], v[:n], hd ** -0.5, seen, dt, up)
        R.check(out[i:i + 1], ref, tol, f"{name}, row {i}")


def _randn(shape, seed, dt):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dt)


@pytest.mark.parametrize("hq,hkv,hd,T,dt", [(2, 1, 64, 100003, BF), (4, 2, 256, 40001, FP)])
def test_a_long_prompt(hq, hkv, hd, T, dt):
    from qwen35_amd.kernels import attention as A
    q, k, v = _randn((T, hq, hd), 1, dt), _randn((T, hkv, hd), 2, dt), _randn((T, hkv, hd), 3, dt)
    out = torch.empty_like(q)
    A.attn_prompt(q, k, v, torch.tensor([0, T], dtype=torch.int32, device="cuda"), out)
    assert out.isfinite().all()
    _rows(out, q, k, v, [0, 1, 31, 32, 127, 5000, T // 2, T - 33, T - 2, T - 1], lambda i: i + 1, dt, "long prompt")


@pytest.mark.parametrize("int8", [False, True])
def test_a_million_keys(int8):
    """A chunk of a prompt and a decode step over 2^20 + 7 keys."""
    from qwen35_amd.kernels import attention as A
    n, page, hd = (1 << 20) + 7, 256, 64
    pages = -(-n // page)
    c = R.cache(pages, page, 1, hd, BF, 5, int8)
    g = torch.Generator(device="cuda").manual_seed(6)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None]
    kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
    k, v = R.gathered(c, table, 0, n)
    q = _randn((20, 4, hd), 7, BF)
    out = torch.empty_like(q)
    A.attn_prompt_paged(q, c[0], c[1], table, kv_len, torch.tensor([0, 20], dtype=torch.int32, device="cuda"), out,
                        k_s=c[2], v_s=c[3])
    _rows(out, q, k, v, [0, 9, 19], lambda i: n - 19 + i, BF, "chunk")
    one = torch.empty_like(q[:1])
    A.attn_decode(q[:1], c[0], c[1], table, kv_len, one, k_s=c[2], v_s=c[3])
    _rows(one, q[:1], k, v, [0], lambda i: n, BF, "decode", 2.0 ** -16 if int8 else None)


def test_thousands_of_sequences():
    from qwen35_amd.kernels import attention as A
    B, page, hq, hkv, hd = 5000, 16, 4, 2, 64
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 60, (B,), generator=g)
    lens[17] = 4000
    need = (lens + page - 1) // page
    pages = int(need.sum())
    table = torch.full((B, int(need.max())), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    for b, m in enumerate(need.tolist()):
        table[b, :m] = order[at:at + m]
        at += m
    table, kv_len = table.cuda(), lens.to(torch.int32).cuda()
    c = R.cache(pages, page, hkv, hd, BF, 9)
    q = _randn((B, hq, hd), 10, BF)
    out = torch.full_like(q, 7)
    A.attn_decode(q, c[0], c[1], table, kv_len, out)
    assert (out[kv_len == 0] == 0).all() and out.isfinite().all()
    for b in (0, 1, 17, 63, 64, 65, 2500, 4936, B - 1):
        k, v = R.gathered(c, table, b, int(lens[b]))
        _rows(out[b:b + 1], q[b:b + 1], k, v, [0], lambda i: k.shape[0], BF, f"sequence {b}")
    # the same lengths as packed prompts
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32).cuda()
    T = int(lens.sum())
    q, k, v = _randn((T, hq, hd), 11, BF), _randn((T, hkv, hd), 12, BF), _randn((T, hkv, hd), 13, BF)
    out = torch.empty_like(q)
    A.attn_prompt(q, k, v, cu, out)
    assert out.isfinite().all()
    for b in (0, 1, 17, 63, 64, 65, 2500, 4936, B - 1):
        a, n = int(cu[b]), int(lens[b])
        if n:
            _rows(out[a:a + n], q[a:a + n], k[a:a + n], v[a:a + n], {0, n // 2, n - 1}, lambda i: i + 1, BF, f"prompt {b}")


def test_one_page_in_many_rows_of_the_table():
    """Sequences that share their first pages, and a table whose rows are one row."""
    from qwen35_amd.kernels import attention as A
    c = R.cache(8, 64, 2, 128, BF, 14)
    table = torch.tensor([[3, 1, 5, 0]], dtype=torch.int32, device="cuda").expand(6, 4)
    lens = [1, 64, 65, 200, 256, 0]
    kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = _randn((6, 8, 128), 15, BF)
    out = torch.empty_like(q)
    A.attn_decode(q, c[0], c[1], table, kv_len, out)
    for b, n in enumerate(lens):
        k, v = R.gathered(c, table, b, n)
        _rows(out[b:b + 1], q[b:b + 1], k, v, [0], lambda i: n, BF, f"sequence {b}")
