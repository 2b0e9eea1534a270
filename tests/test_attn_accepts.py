"""CPU tests of calls that the attention operators' checks let through, and of the lines next to them: what
would be launched is recorded, nothing runs."""
from __future__ import annotations

import pytest

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
