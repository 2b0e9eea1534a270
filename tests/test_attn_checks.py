"""CPU tests of the attention operators' boundary: libqlin.so exports what
include/qlin_attn.h declares, every refusal comes with its status before anything is
launched (the pointers here lead nowhere), and the Python calls check shapes and types."""
from __future__ import annotations

import ctypes
import pathlib
import re

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "qlin_attn.h"
FAKE = 0x10000
BF = torch.bfloat16


@pytest.fixture(scope="module")
def A():
    from qwen35_amd.kernels import attention
    return attention


_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class PagedKV(ctypes.Structure):
    """include/qlin_attn.h qlin_paged_kv."""
    _fields_ = [(f, t) for x in ("k", "v", "k_s", "v_s")
                for f, t in ((x, _P), (x.replace("_", "") + "_page", _L), (x.replace("_", "") + "_token", _L),
                             (x.replace("_", "") + "_head", _L))] + [("dtype", _I), ("num_pages", _I), ("page", _I)]


class Rope(ctypes.Structure):
    """include/qlin_attn.h qlin_rope."""
    _fields_ = [
        ("q", _P), ("q_token", _L), ("q_head", _L), ("k", _P), ("k_token", _L), ("k_head", _L), ("v", _P),
        ("v_token", _L), ("v_head", _L), ("q_out", _P), ("qo_token", _L), ("qo_head", _L), ("k_out", _P),
        ("ko_token", _L), ("ko_head", _L), ("slots", _P), ("slots_64", _I), ("pos", _P), ("pos_axis", _L),
        ("pos_token", _L), ("pos_64", _I), ("freqs", _P), ("freqs_64", _I), ("q_w", _P), ("k_w", _P), ("w_dtype", _I),
        ("one_plus", _I), ("eps", _F), ("T", _I), ("q_heads", _I), ("kv_heads", _I), ("hd", _I), ("rot", _I),
        ("axes", _I), ("sections", _I * 3), ("interleaved", _I), ("dtype", _I),
    ]


def _lib(A):
    """The library with this file's own view of the ABI (structs by address)."""
    from qwen35_amd.kernels import qlin
    L = ctypes.CDLL(str(qlin.LIB_PATH))
    L.qlin_last_error.restype = ctypes.c_char_p
    for n, sig in A._SIGS.items():
        getattr(L, n).argtypes = [_P if t is ctypes.c_char_p else t for t in sig]
        getattr(L, n).restype = ctypes.c_int
    return qlin, L


def test_packed_structs_are_the_headers(A):
    """The packing formats give the fields the places that a C compiler does."""
    assert A._PAGED_KV.size == ctypes.sizeof(PagedKV) and A._ROPE.size == ctypes.sizeof(Rope)
    kv = PagedKV.from_buffer_copy(A._PAGED_KV.pack(*range(1, 20)))
    assert [getattr(kv, f) for f, _ in PagedKV._fields_] == list(range(1, 20))
    vals = list(range(1, 40))
    r = Rope.from_buffer_copy(A._ROPE.pack(*vals))
    got = []
    for f, _ in Rope._fields_:
        x = getattr(r, f)
        got += list(x) if f == "sections" else [x]
    assert got[:len(vals)] == vals and len(got) == len(vals)


def test_header_and_library_agree(A):
    names = re.findall(r"^int (qlin_\w+)\s*\(", HEADER.read_text(), re.M)
    assert set(names) == set(A.EXPORTS) and len(names) == 4
    _, L = _lib(A)
    for n in names:
        assert hasattr(L, n)


def _kv(A, **kw):
    d = dict(k=FAKE, k_page=64 * 256, k_token=256, k_head=64, v=FAKE, v_page=64 * 256, v_token=256, v_head=64,
             dtype=2, num_pages=8, page=64)
    d.update(kw)
    return PagedKV(**d)


def _kv8(A, **kw):
    d = dict(dtype=4, k_s=FAKE, ks_page=256, ks_token=4, ks_head=1, v_s=FAKE, vs_page=256, vs_token=4, vs_head=1)
    d.update(kw)
    return _kv(A, **d)


DECODE = dict(q=FAKE, qs=512, qh=64, kv=None, table=FAKE, ts=8, mp=8, kv_len=FAKE, out=FAKE + 4096, os=512, oh=64, B=2, hq=8,
              hkv=4, hd=64, dt=2, scale=0.125, ws=FAKE, nws=256 << 20, st=None)


def _decode(A, **kw):
    qlin, L = _lib(A)
    d = dict(DECODE, kv=ctypes.byref(_kv(A)))
    d.update(kw)
    return L.qlin_attn_decode(*d.values()), L.qlin_last_error().decode()


@pytest.mark.parametrize("bad,text", [
    (dict(B=-1), "negative"), (dict(hq=9), "multiple"), (dict(hkv=0), "multiple"), (dict(hq=260), "more than 64"),
    (dict(hd=96), "head size"), (dict(dt=3), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=None), "null q"), (dict(q=FAKE + 2), "q must be 16-byte"),
    (dict(qs=511), "multiples of 8"), (dict(out=None), "null out"), (dict(os=0), "overlap"), (dict(oh=8), "overlap"),
    (dict(table=None), "null page table"), (dict(kv_len=None), "null page table"), (dict(kv_len=FAKE + 2), "4-byte"),
    (dict(mp=-1), "negative"), (dict(mp=1 << 28), "keys a sequence"), (dict(ws=None), "workspace"),
    (dict(nws=1 << 20), "workspace"), (dict(ws=FAKE + 8), "256-byte"), (dict(B=1 << 24), "more than"),
    (dict(B=(1 << 16) + 1), "more than 65536 sequences"), (dict(hq=1 << 17, hkv=1 << 16), "more than 65536 query heads"),
    (dict(B=1 << 16, hq=512, hkv=512), "too many rows"), (dict(qs=1 << 30), "above"), (dict(out=FAKE), "must not be q"),
])
def test_decode_refusals(A, bad, text):
    rc, msg = _decode(A, **bad)
    assert rc < 0 and text in msg, (rc, msg)


@pytest.mark.parametrize("bad,text", [
    (dict(page=48), "power of two"), (dict(page=8), "power of two"), (dict(page=2048), "power of two"),
    (dict(num_pages=0), "no pages"), (dict(dtype=1), "cache dtype"), (dict(k=None), "null k_cache"),
    (dict(v=FAKE + 8), "v_cache must be 16-byte"), (dict(k_token=260), "multiples of 8"),
    (dict(v_page=4), "page strides"), (dict(k_s=FAKE), "no scales"), (dict(k_page=1 << 31), "page strides above"),
])
def test_cache_refusals(A, bad, text):
    rc, msg = _decode(A, kv=ctypes.byref(_kv(A, **bad)))
    assert rc < 0 and text in msg, (rc, msg)


@pytest.mark.parametrize("bad,text", [
    (dict(k_s=None), "needs k_s"), (dict(v_s=FAKE + 2), "4-byte"), (dict(vs_head=-1), "negative"), (dict(ks_page=1 << 30), "too large"),
    (dict(k_token=264), "multiples of 16"),
])
def test_int8_cache_refusals(A, bad, text):
    rc, msg = _decode(A, kv=ctypes.byref(_kv8(A, **bad)))
    assert rc < 0 and text in msg, (rc, msg)


def test_nothing_to_do_is_no_launch(A):
    assert _decode(A, B=0)[0] == 0
    qlin, L = _lib(A)
    assert L.qlin_attn_prompt(*([None, 0, 0] * 3), None, None, None, 0, 0, 0, 0, 0, 8, 4, 64, 2, 0.125, 1, None, 0,
                              None) == 0
    assert L.qlin_attn_prompt_paged(None, 0, 0, None, None, 0, 0, None, None, None, 0, 0, 0, 3, 8, 4, 64, 2, 0.125, 1,
                                    None, 0, None) == 0


PROMPT = dict(q=FAKE, qt=512, qh=64, k=FAKE, kt=256, kh=64, v=FAKE, vt=256, vh=64, cu=FAKE, ck=FAKE, out=FAKE + 4096, ot=512,
              oh=64, T=9, Tk=9, B=2, hq=8, hkv=4, hd=64, dt=2, scale=0.125, causal=1, ws=FAKE, nws=256 << 20, st=None)


@pytest.mark.parametrize("bad,text", [
    (dict(T=-1), "negative"), (dict(T=1 << 25), "more than"), (dict(cu=None), "null row bounds"),
    (dict(ck=FAKE + 1), "4-byte"), (dict(k=None), "null k"), (dict(v=FAKE + 4), "v must be 16-byte"),
    (dict(ot=8), "rows of out overlap"), (dict(ws=None), "workspace"), (dict(hd=32), "head size"),
    (dict(scale=-1.0), "scale"), (dict(kt=1 << 27), "above"), (dict(B=(1 << 16) + 1), "more than 65536 sequences"),
    (dict(T=(1 << 24) - 1, hq=512, hkv=8), "too many rows"),
])
def test_prompt_refusals(A, bad, text):
    qlin, L = _lib(A)
    d = dict(PROMPT)
    d.update(bad)
    rc = L.qlin_attn_prompt(*d.values())
    assert rc < 0 and text in L.qlin_last_error().decode(), (rc, L.qlin_last_error())


def _rope(A, cache=None, **kw):
    qlin, L = _lib(A)
    d = dict(q=FAKE, q_token=512, q_head=64, k=FAKE, k_token=256, k_head=64, v=FAKE, v_token=256, v_head=64,
             q_out=FAKE, qo_token=512, qo_head=64, k_out=FAKE, ko_token=256, ko_head=64, slots=FAKE, pos=FAKE,
             pos_axis=4, pos_token=1, freqs=FAKE, q_w=FAKE, k_w=FAKE, w_dtype=2, one_plus=1, eps=1e-6, T=4, q_heads=8,
             kv_heads=4, hd=64, rot=64, axes=1, sections=(32, 0, 0), interleaved=0, dtype=2)
    d.update(kw)
    d["sections"] = (ctypes.c_int * 3)(*d["sections"])
    return (L.qlin_qk_norm_rope(ctypes.byref(Rope(**d)), ctypes.byref(cache) if cache is not None else None, None),
            L.qlin_last_error().decode())


@pytest.mark.parametrize("bad,text", [
    (dict(T=-3), "negative"), (dict(rot=24), "rotated"), (dict(rot=80), "rotated"), (dict(axes=4), "axes"),
    (dict(sections=(30, 0, 0)), "add up"), (dict(axes=2, sections=(33, -1, 0)), "negative section"),
    (dict(axes=3, interleaved=1, sections=(8, 12, 12)), "no 12 turns"), (dict(k_out=None), "neither"),
    (dict(pos=None), "null positions"), (dict(freqs=FAKE + 4, freqs_64=1), "aligned"), (dict(w_dtype=7), "weight"),
    (dict(q_out=None), "null q_out"), (dict(qo_head=0), "overlap"), (dict(ko_token=8), "overlap"),
    (dict(cache=1, v=None), "values and slots"), (dict(cache=1, slots=None), "values and slots"),
    (dict(cache=1, slots=FAKE + 4, slots_64=1), "aligned"), (dict(T=1 << 25), "more than"),
])
def test_rope_refusals(A, bad, text):
    bad = dict(bad)
    rc, msg = _rope(A, _kv(A) if bad.pop("cache", None) else None, **bad)
    assert rc < 0 and text in msg, (rc, msg)


@pytest.mark.parametrize("bad,text", [(dict(k_token=0), "overlap"), (dict(v_page=8), "pages of the cache overlap")])
def test_rope_refuses_a_cache_that_overlaps_itself(A, bad, text):
    rc, msg = _rope(A, _kv(A, **bad))
    assert rc < 0 and text in msg, (rc, msg)
    rc, msg = _rope(A, _kv8(A, ks_token=0))
    assert rc < 0 and "scales of the cache overlap" in msg, (rc, msg)


def _t(*shape, dt=BF):
    return torch.zeros(shape, dtype=dt)


def test_python_checks(A):
    q, out = _t(2, 8, 64), _t(2, 8, 64)
    kc, vc = _t(4, 16, 4, 64), _t(4, 16, 4, 64)
    table, n = _t(2, 3, dt=torch.int32), _t(2, dt=torch.int32)
    ok = dict(q=q, k_cache=kc, v_cache=vc, table=table, kv_len=n, out=out)
    for bad, text in [
        (dict(), "must be on the GPU"), (dict(q=_t(2, 8, 64, dt=torch.float32)), "bfloat16 or float16"),
        (dict(q=_t(2, 512)), "rows, heads, hd"), (dict(out=_t(3, 8, 64)), "2 rows"),
        (dict(out=_t(2, 8, 64, dt=torch.float16)), "out must be torch.bfloat16"),
        (dict(k_cache=_t(4, 16, 4, 128)), "both be"), (dict(table=_t(3, 3, dt=torch.int32)), "table must be"),
        (dict(table=_t(2, 3, dt=torch.int64)), "int32"), (dict(kv_len=_t(3, dt=torch.int32)), "kv_len must be"),
        (dict(k_cache=_t(4, 16, 4, 64, dt=torch.int8), v_cache=_t(4, 16, 4, 64, dt=torch.int8)), "needs its scales"),
        (dict(k_s=_t(4, 16, 4, dt=torch.float32)), "no scales"),
        (dict(k_cache=_t(4, 16, 4, 64, dt=torch.float16), v_cache=_t(4, 16, 4, 64, dt=torch.float16)), "int8 or"),
        (dict(q=_t(2, 8, 128)[..., ::2]), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            A.attn_decode(**dict(ok, **bad))
    cu = _t(3, dt=torch.int32)
    with pytest.raises(ValueError, match="cu_k"):
        A.attn_prompt(q, _t(5, 4, 64), _t(5, 4, 64), cu, out)
    with pytest.raises(ValueError, match="both be"):
        A.attn_prompt(q, _t(2, 4, 64), _t(2, 2, 64), cu, out)
    with pytest.raises(ValueError, match="table must be"):
        A.attn_prompt_paged(q, kc, vc, table, n, _t(2, dt=torch.int32), out)
    k, pos, fr = _t(2, 4, 64), _t(2, dt=torch.int64), _t(16, dt=torch.float32)
    for bad, text in [
        (dict(), "give k_out"), (dict(k_out=k, pos=_t(3, 2, dt=torch.int64)), "need sections"),
        (dict(k_out=k, pos=_t(3, 2, dt=torch.int64), sections=(8, 8)), "one length"),
        (dict(k_out=k, pos=_t(3, dt=torch.int64)), "pos must be"), (dict(k_out=k, pos=_t(2)), "int32 or int64"),
        (dict(k_out=k, freqs=_t(16)), "float32 or float64"), (dict(k_out=k, q_w=_t(32)), "q_w must be"),
        (dict(k_cache=kc, v_cache=vc, v=k), "slots"), (dict(k_out=_t(2, 3, 64)), "k_out must be"),
        (dict(k_cache=kc, v_cache=vc, v=k, slots=_t(3, dt=torch.int64)), "slots must be"),
    ]:
        d = dict(q=q, k=k, pos=pos, freqs=fr, q_out=out)
        d.update(bad)
        with pytest.raises(ValueError, match=text):
            A.qk_norm_rope(**d)
