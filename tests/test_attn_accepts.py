"""CPU tests of calls that the attention operators' checks let through, and of the lines next to them: what
would be launched is recorded, nothing runs."""
from __future__ import annotations

import pytest
import torch

import attn_dispatch as D


@pytest.fixture(scope="module")
def tmp(tmp_path_factory):
    return tmp_path_factory.mktemp("fake")


def _accepted(tmp, *calls):
    for call, (status, launches, msg) in zip(calls, D.run(tmp, calls)):
        assert status == 0 and launches, (call, msg)


def _refused(tmp, text, *calls):
    for call, (status, launches, msg) in zip(calls, D.run(tmp, calls)):
        assert status < 0 and not launches and text in msg, (call, status, msg)


def test_plain_calls(tmp):
    kv, kv8 = D.cache(4, 64), D.cache(4, 64, dtype=D.I8)
    _accepted(tmp, D.decode(kv), D.decode(kv8), D.paged(kv), D.paged(kv8), D.prompt(), D.rope(), D.rope(kv), D.rope(kv8))


def _head_major(pages, page, hd, dtype=D.BF16):
    """A cache whose heads lie apart, [heads][pages][page][hd]."""
    far = pages * page * hd
    kw = dict(k_page=page * hd, k_token=hd, k_head=far, v_page=page * hd, v_token=hd, v_head=far)
    if dtype == D.I8:
        kw |= dict(ks_page=page, ks_token=1, ks_head=pages * page, vs_page=page, vs_token=1, vs_head=pages * page)
    return D.cache(4, hd, pages, page, dtype, **kw)


def test_heads_that_lie_far_apart(tmp):
    for dtype in (D.BF16, D.I8):
        kv = _head_major(1 << 15, 64, 256, dtype)  # 2^29 elements a head
        _accepted(tmp, D.decode(kv, hd=256), D.paged(kv, hd=256), D.rope(kv, hd=256))
    far = 1 << 30
    _accepted(tmp, D.prompt(qh=far, qt=64, kh=far, kt=64, vh=far, vt=64, oh=far, ot=64),
              D.rope(q_head=far, q_token=64, k_head=far, k_token=64, qo_head=far, qo_token=64, ko_head=far, ko_token=64))
    over = 1 << 31
    _refused(tmp, "stride", D.decode(D.cache(4, 64, k_head=over)), D.prompt(oh=over), D.rope(q_head=over),
             D.decode(D.cache(4, 64, dtype=D.I8, vs_head=1 << 30)), D.decode(D.cache(4, 64, v_token=1 << 27)))


def test_strides_of_an_axis_of_one(tmp):
    """They are never used: any number will do."""
    for s in (1, 3, -8, 1 << 40):
        one = D.cache(1, 64, pages=1, k_head=s, v_head=s, k_page=s, v_page=s)
        _accepted(tmp, D.decode(one, B=1, hkv=1, qs=s, os=s), D.paged(one, T=1, B=1, hkv=1, qt=s, ot=s),
                  D.prompt(T=1, B=1, hkv=1, hq=1, qt=s, qh=s, kt=s, kh=s, vt=s, vh=s, ot=s, oh=s),
                  D.rope(one, T=1, hkv=1, q_token=s, k_token=s, k_head=s, v_token=s, v_head=s, qo_token=s, ko_token=s,
                         ko_head=s))
        one8 = D.cache(1, 64, pages=1, dtype=D.I8, ks_head=s, vs_head=s, ks_page=s, vs_page=s)
        _accepted(tmp, D.decode(one8, B=1, hkv=1), D.rope(one8, T=1, hkv=1))
    two = D.cache(2, 64, k_head=65)
    _refused(tmp, "multiples of 8", D.decode(two, hkv=2), D.prompt(qt=513), D.rope(ko_token=129))


def test_a_table_of_no_pages(tmp):
    """All sequences are empty; torch gives such a table the address 0."""
    kv = D.cache(4, 64)
    _accepted(tmp, D.decode(kv, table=None, max_pages=0), D.paged(kv, table=None, max_pages=0))
    _refused(tmp, "null page table", D.decode(kv, table=None), D.paged(kv, table=None),
             D.decode(kv, table=None, max_pages=0, kv_len=None))


def test_outputs_next_to_inputs(tmp):
    """Columns of one buffer's rows, in any order, and the planes of one cache."""
    row = 8 * 128 + 2 * 4 * 64            # heads of a query and a gate, keys, values
    k0 = D.Q + 2 * 8 * 128
    _accepted(tmp,
              D.prompt(qt=row, qh=128, k=k0, kt=row, v=k0 + 2 * 256, vt=row, out=D.Q + 2 * 64, ot=row, oh=128),
              D.prompt(out=D.Q + 9 * 512 * 2), D.prompt(out=D.K - 9 * 512 * 2), D.decode(D.cache(4, 64), out=D.Q + 2048),
              # q_out and k_out in place, or q_out in the gates' columns
              D.rope(q_token=row, q_head=128, q_out=D.Q, qo_token=row, qo_head=128, k=k0, k_token=row, k_out=k0,
                     ko_token=row, v=k0 + 512, v_token=row),
              D.rope(q_token=row, q_head=128, q_out=D.Q + 128, qo_token=row, qo_head=128, k=k0, k_token=row),
              # keys and values of a page next to each other, or of a token, or of a head
              D.rope(D.cache(4, 64, v=D.K + 2 * 64 * 256, k_page=2 * 64 * 256, v_page=2 * 64 * 256)),
              D.rope(D.cache(4, 64, v=D.K + 2 * 256, k_page=128 * 256, k_token=512, v_page=128 * 256, v_token=512)),
              D.rope(D.cache(4, 64, v=D.K + 2 * 64, k_page=128 * 256, k_token=512, k_head=128, v_page=128 * 256,
                             v_token=512, v_head=128)))


def test_outputs_that_lie_in_inputs(tmp):
    kv, kv8 = D.cache(4, 64), D.cache(4, 64, dtype=D.I8)
    _refused(tmp, "out overlaps q", D.prompt(out=D.Q + 512 * 2), D.prompt(out=D.Q - 2 * 512 * 2 + 16),
             D.decode(kv, out=D.Q + 1024), D.paged(kv, out=D.Q + 16))
    _refused(tmp, "out overlaps k", D.prompt(out=D.K), D.prompt(out=D.K + 256), D.paged(kv, out=D.K + (1 << 17)),
             D.decode(kv8, out=D.K))
    _refused(tmp, "out overlaps v", D.prompt(out=D.V + 128 * 4), D.decode(kv, out=D.V))
    _refused(tmp, "out overlaps k_s", D.decode(kv8, out=D.KS + 512))
    _refused(tmp, "overlaps q", D.rope(q_out=D.Q + 1024), D.rope(q_out=D.Q, qo_token=1024), D.rope(k_out=D.Q))
    _refused(tmp, "overlaps k", D.rope(q_out=D.K), D.rope(k_out=D.K + 512), D.rope(k_out=D.K, ko_token=512))
    _refused(tmp, "overlaps v", D.rope(kv, k_out=D.V + (1 << 43)), D.rope(kv, q_out=D.V + (1 << 43) + 64))
    _refused(tmp, "overlaps q_out", D.rope(k_out=D.OUT + 128))
    _refused(tmp, "overlaps v_cache", D.rope(D.cache(4, 64, k=D.V)), D.rope(D.cache(4, 64, k=D.V + 256)))
    _refused(tmp, "overlaps v_s", D.rope(D.cache(4, 64, dtype=D.I8, k_s=D.VS)))
    _refused(tmp, "overlaps k_cache", D.rope(kv, q=D.K), D.rope(kv, k_out=D.K + 4096))


def test_overlaps_are_found_as_by_counting(tmp):
    """Random layouts of a few rows and heads: refused where some byte belongs to both, and only there."""
    import random
    rng = random.Random(5)
    calls, want = [], []
    while len(calls) < 400:
        B, hq, hkv = rng.randint(1, 4), rng.choice([1, 2, 4]), 1
        row = [64 * rng.randint(1, 9) + rng.choice([0, 0, 8, 24]) for _ in range(2)]
        head = [64 * rng.randint(1, 9) + rng.choice([0, 0, 8, 40]) for _ in range(2)]
        if rng.random() < 0.5:
            row[1], head[1] = row[0], head[0]
        at = 8 * rng.randint(-300, 300)
        a, b = ({o + b * r + h * s + e for b in range(B) for h in range(hq) for e in range(64)}
                for o, r, s in ((0, row[0], head[0]), (at, row[1], head[1])))
        if at == 0 or len(b) != B * hq * 64:
            continue
        calls.append(D.decode(D.cache(hkv, 64), B=B, hq=hq, hkv=hkv, qs=row[0], qh=head[0], out=D.Q + 2 * at, os=row[1],
                              oh=head[1]))
        want.append(bool(a & b))
    assert 40 < sum(want) < 360
    for call, bad, (status, launches, msg) in zip(calls, want, D.run(tmp, calls)):
        assert (status < 0 and "out overlaps q" in msg and not launches) if bad else (status == 0 and launches), (call, msg)


def test_outputs_that_overlap_themselves(tmp):
    """Strides that are each long enough, but lead to the same place in two ways."""
    _refused(tmp, "rows of out overlap", D.prompt(ot=64, oh=64), D.prompt(ot=64, oh=256), D.prompt(ot=128, oh=192),
             D.decode(D.cache(4, 64), os=64, oh=64), D.paged(D.cache(4, 64), ot=512, oh=72 * 64 + 8 - 4 * 512))
    _refused(tmp, "rows of q_out overlap", D.rope(qo_token=64, qo_head=64))
    _refused(tmp, "rows of k_out overlap", D.rope(ko_token=128, ko_head=192))
    _refused(tmp, "rows of k_cache overlap", D.rope(D.cache(4, 64, k_page=64 * 128)), D.rope(D.cache(4, 64, k_token=64)))
    _refused(tmp, "rows of v_s overlap", D.rope(D.cache(4, 64, dtype=D.I8, vs_token=2)))
    # heads before tokens, tokens before pages, gaps
    _accepted(tmp, D.prompt(ot=64, oh=9 * 64), D.prompt(ot=192, oh=9 * 192 + 8), D.prompt(T=2, hq=4, ot=192, oh=2 * 192),
              D.rope(D.cache(4, 64, k_page=64, k_token=8 * 64, k_head=8 * 64 * 64)),
              D.rope(D.cache(4, 64, dtype=D.I8, vs_page=1, vs_token=8, vs_head=512)), D.prompt(T=2, hq=4, ot=192, oh=128))


def test_overlaps_within_are_found_as_by_counting(tmp):
    import random
    rng = random.Random(6)
    calls, want = [], []
    for _ in range(400):
        T, hq = rng.randint(1, 6), rng.choice([1, 2, 4, 8])
        row, head = (64 + 8 * rng.randint(0, 70) for _ in range(2))
        runs = [t * row + h * head for t in range(T) for h in range(hq)]
        calls.append(D.prompt(T=T, hq=hq, hkv=1, B=1, ot=row, oh=head))
        want.append(len({o + e for o in runs for e in range(0, 64, 8)}) < len(runs) * 8)
    assert 40 < sum(want) < 360
    for call, bad, (status, launches, msg) in zip(calls, want, D.run(tmp, calls)):
        assert (status < 0 and "rows of out overlap" in msg and not launches) if bad else (status == 0 and launches), (call, msg)


def test_sizes_past_32_bits_are_refused():
    """A ctypes int keeps the low 32 bits of what it is given: 2^32 + 5 rows would be 5."""
    from qwen35_amd.kernels import attention as A
    far = (1 << 32) + 5

    def t(*shape, dt=torch.bfloat16):
        return torch.empty(shape, dtype=dt, device="meta")

    q, k, kv, n, cu = t(2, 8, 64), t(2, 4, 64), t(4, 16, 4, 64), t(2, dt=torch.int32), t(3, dt=torch.int32)
    table = t(2, 3, dt=torch.int32)
    for call in (lambda: A.attn_prompt(q, t(far, 4, 64), t(far, 4, 64), cu, q, cu_k=cu),
                 lambda: A.attn_prompt(t(far, 8, 64), k, k, cu, t(far, 8, 64), cu_k=cu),
                 lambda: A.attn_prompt(q, k, k, t(far, dt=torch.int32), q),
                 lambda: A.attn_decode(t(far, 8, 64), kv, kv, table, n, t(far, 8, 64)),
                 lambda: A.attn_decode(q, t(far, 16, 4, 64), t(far, 16, 4, 64), table, n, q),
                 lambda: A.attn_decode(q, kv, kv, t(2, far, dt=torch.int32), n, q),
                 lambda: A.attn_prompt_paged(q, kv, kv, t(2, far, dt=torch.int32), n, cu, q),
                 lambda: A.qk_norm_rope(t(far, 8, 64), t(far, 4, 64), t(far, dt=torch.int64),
                                        t(16, dt=torch.float32), t(far, 8, 64), t(far, 4, 64))):
        with pytest.raises(ValueError, match="is more than"):
            call()
