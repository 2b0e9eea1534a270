"""CPU tests of calls of a step of several candidates that the checks let through, and of the lines next to them: what
would be launched is recorded, nothing runs."""
from __future__ import annotations

import attn_dispatch as D
import pytest

U, TEMP, LOGP, PTABLE, PLEN = ((i + 21) << 44 for i in range(5))


@pytest.fixture(scope="module")
def tmp(tmp_path_factory):
    return tmp_path_factory.mktemp("fake")


def shared(kv, B=8, G=1, hq=8, hkv=4, hd=64, ppages=8, pages=8, dt=D.BF16, **kw):
    d = dict(q=D.Q, qs=hq * hd, qh=hd, kv=kv, ptable=PTABLE, ps=ppages, pp=ppages, plen=PLEN, cu=D.CU, G=G, table=D.TABLE,
             ts=pages, mp=pages, kv_len=D.LEN, out=D.OUT, os=hq * hd, oh=hd, B=B, hq=hq, hkv=hkv, hd=hd, dt=dt, scale=0.125,
             ws=D.WS, nws=256 << 20, st=None)
    return ["qlin_attn_decode_shared", *(d | kw).values()]


def sample(B=1, V=1000, k=20, dt=3, **kw):
    d = dict(x=D.Q, dt=dt, xs=V, B=B, V=V, k=k, u=U, temp=None, t=1.0, pp=None, p=1.0, mp=None, m=0.0, tokens=D.OUT, t64=1,
             logp=LOGP, ws=D.WS, nws=256 << 20, st=None)
    return ["qlin_sample", *(d | kw).values()]


def _run(tmp, call, launches):
    status, got, msg = D.run(tmp, [call])[0]
    assert status == 0 and len(got) == launches, (call, got, msg)
    return got


def _refused(tmp, text, *calls):
    for call, (status, launches, msg) in zip(calls, D.run(tmp, calls)):
        assert status < 0 and not launches and text in msg, (call, status, msg)


@pytest.mark.parametrize("B,hq,hkv,hd,i8,ppages,form", [
    (1, 8, 2, 256, 0, 3, 1), (4, 8, 2, 256, 0, 2000, 1), (8, 8, 2, 256, 0, 8, 1), (8, 8, 2, 256, 0, 2000, 2),
    (8, 8, 2, 256, 1, 2000, 1), (9, 8, 2, 256, 0, 8, 0), (1, 17, 1, 64, 0, 8, 0), (1, 64, 1, 128, 1, 8, 0),
    (2, 16, 1, 128, 0, 2000, 2), (33, 3, 3, 128, 0, 8, 0), (32, 3, 3, 128, 0, 8, 1)])
@pytest.mark.parametrize("dt", [D.BF16, D.F16])
def test_forms(tmp, B, hq, hkv, hd, i8, ppages, form, dt):
    """Rows of a key head up to 16 take one tile; up to 32 two where the prefix's bytes by its table are many; others,
    and more than 16 query heads to a key head, the wide form."""
    kv = D.cache(hkv, hd, pages=4096, dtype=D.I8 if i8 else dt)
    got = _run(tmp, shared(kv, B, 1, hq, hkv, hd, ppages, dt=dt), 2)
    assert "13shared_kernelI" in got[0][0] and f"Li{hd}ELb{i8}ELi{form}E" in got[0][0], got
    assert "shared_join" in got[1][0]


def test_largest(tmp):
    kv = D.cache(1, 64, pages=1 << 20)
    for call in (shared(kv, 1 << 14, 1 << 14, 1, 1, 64), shared(kv, 4096, 1, 64, 1, 64, ppages=1 << 17),
                 shared(kv, 1, 3, 1, 1, 64, pages=1 << 17), shared(kv, 5, 1, 5, 1, 64, ppages=0, pages=0, table=None, ptable=None)):
        got = _run(tmp, call, 2)
        assert all(0 < g < 1 << 24 for _, g in got), got
    _run(tmp, shared(kv, 0, 1, 1, 1), 0)
    _run(tmp, shared(kv, 1, 0, 1, 1), 0)
    # (B x query heads x hd past what the workspace holds sums of)
    _refused(tmp, "workspace holds", shared(kv, 1 << 14, 1, 64, 1, 64))
    _refused(tmp, "null", shared(kv, 1, 1, 1, 1, cu=None), shared(kv, 1, 1, 1, 1, ptable=None), shared(kv, 1, 1, 1, 1, plen=None))


def test_shared_overlaps(tmp):
    kv = D.cache(4, 64)
    _refused(tmp, "overlap", shared(kv, out=D.K + 64), shared(kv, out=D.Q + 1024))
    _refused(tmp, "out must not be q", shared(kv, out=D.Q))
    _run(tmp, shared(kv, q=D.K, out=D.OUT), 2)  # (reading twice is no overlap)


@pytest.mark.parametrize("B,V,k,chunks", [(1, 1, 1, 1), (1, 8192, 20, 1), (1, 8193, 20, 2), (1, 248320, 20, 31), (64, 248320, 50, 16),
                                          (1, 248320, 128, 31), (1, 1 << 30, 128, 31), (4096, 50021, 128, 7),
                                          (1 << 16, 8193, 128, 2), (1 << 16, 1 << 20, 1, 64),
                                          (8, 248320, 50, 31), (17, 248320, 50, 16), (256, 131072, 20, 16)])
def test_sample_grids(tmp, B, V, k, chunks):
    (name, grid), = _run(tmp, sample(B, V, k), 1)
    assert "sample_kernel" in name and grid == B * chunks < 1 << 24


def test_sample_limits(tmp):
    _run(tmp, sample(B=0), 0)
    _run(tmp, sample(B=5, xs=0), 1)  # one row for all
    _refused(tmp, "top_k", sample(k=0), sample(k=129))
    _refused(tmp, "rows", sample(B=(1 << 16) + 1))
    _refused(tmp, "vocabulary", sample(V=0), sample(V=(1 << 30) + 1))
    _refused(tmp, "overlap", sample(V=1000, tokens=D.Q + 8), sample(B=4, logp=D.OUT + 8), sample(tokens=U, t64=0))
    _refused(tmp, "workspace", sample(ws=None), sample(nws=1 << 20))
    _refused(tmp, "must be from", sample(t=-1.0), sample(p=float("nan")), sample(m=float("inf")))
