"""CPU tests of the boundary of a decode step of several candidates: libqlin.so exports what
include/qlin_candidates.h declares, every refusal comes with its status before anything is launched (the
pointers here lead nowhere), and the Python calls check shapes and types."""
from __future__ import annotations

import ctypes
import pathlib
import re

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "qlin_candidates.h"
FAKE = 0x100000
BF, F32 = torch.bfloat16, torch.float32
_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class PagedKV(ctypes.Structure):
    """include/qlin_attn.h qlin_paged_kv."""
    _fields_ = [(f, t) for x in ("k", "v", "k_s", "v_s")
                for f, t in ((x, _P), (x.replace("_", "") + "_page", _L), (x.replace("_", "") + "_token", _L),
                             (x.replace("_", "") + "_head", _L))] + [("dtype", _I), ("num_pages", _I), ("page", _I)]


class Logits(ctypes.Structure):
    """include/qlin_candidates.h qlin_logits."""
    _fields_ = [("logits", _P), ("logits_row", _L), ("out", _P), ("out_row", _L), ("tokens", _P), ("tokens_row", _L),
                ("lens", _P), ("prompt_lens", _P), ("repetition", _P), ("presence", _P), ("frequency", _P),
                ("bias_ids", _P), ("bias_ids_row", _L), ("bias", _P), ("bias_row", _L), ("mask", _P), ("mask_row", _L),
                ("tokens_64", _I), ("mask_bytes", _I), ("B", _I), ("V", _I), ("history", _I), ("biases", _I),
                ("dtype", _I), ("out_dtype", _I), ("repetition_all", _F), ("presence_all", _F), ("frequency_all", _F)]


@pytest.fixture(scope="module")
def S():
    from qwen35_amd.kernels import sampling
    return sampling


def _lib(S):
    from qwen35_amd.kernels import qlin
    L = ctypes.CDLL(str(qlin.LIB_PATH))
    L.qlin_last_error.restype = ctypes.c_char_p
    for n in S.EXPORTS:
        getattr(L, n).argtypes = [_P if t is ctypes.c_char_p else t for t in S._ALL[n]]
        getattr(L, n).restype = ctypes.c_int
    return L


def test_header_and_library_agree(S):
    names = re.findall(r"^int (qlin_\w+)\s*\(", HEADER.read_text(), re.M)
    assert set(names) == set(S.EXPORTS) and len(names) == 3
    L = _lib(S)
    for n in names:
        assert hasattr(L, n)


def test_packed_struct_is_the_headers(S):
    assert S._LOGITS.size == ctypes.sizeof(Logits)
    got = Logits.from_buffer_copy(S._LOGITS.pack(*range(1, 29)))
    assert [getattr(got, f) for f, _ in Logits._fields_] == list(range(1, 29))


# ------------------------------------------------------------------ the C boundary

def _kv(**kw):
    d = dict(k=FAKE, k_page=64 * 256, k_token=256, k_head=64, v=2 * FAKE, v_page=64 * 256, v_token=256, v_head=64,
             dtype=2, num_pages=8, page=64)
    return PagedKV(**(d | kw))


SHARED = dict(q=4 * FAKE, qs=512, qh=64, kv=None, pt=5 * FAKE, pts=8, pmp=8, plen=5 * FAKE, cu=5 * FAKE, G=1, table=5 * FAKE,
              ts=8, mp=8, kv_len=5 * FAKE, out=6 * FAKE, os=512, oh=64, B=2, hq=8, hkv=4, hd=64, dt=2, scale=0.125,
              ws=8 * FAKE, nws=256 << 20, st=None)


@pytest.mark.parametrize("bad,text", [
    (dict(B=-1), "negative"), (dict(G=-1), "negative"), (dict(hq=9), "multiple"), (dict(hkv=0), "multiple"),
    (dict(hq=260), "more than 64"), (dict(hd=96), "head size"), (dict(dt=3), "dtype"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(q=None), "null q"), (dict(q=4 * FAKE + 2), "q must be 16-byte"),
    (dict(qs=511), "multiples of 8"), (dict(out=None), "null out"), (dict(os=0), "overlap"), (dict(oh=8), "overlap"),
    (dict(table=None), "null page table"), (dict(pt=None), "null page table"), (dict(kv_len=None), "null page table"),
    (dict(plen=None), "null page table"), (dict(plen=FAKE + 2), "4-byte"), (dict(cu=None), "null sequence bounds"),
    (dict(cu=FAKE + 1), "4-byte"), (dict(mp=-1), "negative"), (dict(pmp=-1), "negative"),
    (dict(pmp=1 << 28), "keys a sequence"), (dict(ws=None), "workspace"), (dict(nws=1 << 20), "workspace"),
    (dict(ws=8 * FAKE + 8), "256-byte"), (dict(B=(1 << 16) + 1), "more than 65536 sequences"),
    (dict(G=(1 << 16) + 1), "more than 65536 groups"), (dict(B=1 << 16, out=1 << 40), "more than the workspace"),
    (dict(out=4 * FAKE), "must not be q"), (dict(out=4 * FAKE + 128), "overlaps q"), (dict(out=FAKE + 1024), "overlaps k_cache"),
    (dict(out=2 * FAKE + 1024), "overlaps v_cache"), (dict(nws=(5 << 20) + 4096), "more than the workspace"),
])
def test_shared_refusals(S, bad, text):
    L = _lib(S)
    rc = L.qlin_attn_decode_shared(*(SHARED | dict(kv=ctypes.byref(_kv())) | bad).values())
    assert rc < 0 and text in L.qlin_last_error().decode(), L.qlin_last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=1), "cache dtype"), (dict(page=48), "page of 48"), (dict(num_pages=0), "no pages"), (dict(k=None), "null k_cache"),
    (dict(dtype=4, k_head=64, k_token=256), "needs k_s"), (dict(k_s=FAKE), "has no scales"), (dict(k_page=4), "page strides"),
])
def test_shared_cache_refusals(S, bad, text):
    L = _lib(S)
    rc = L.qlin_attn_decode_shared(*(SHARED | dict(kv=ctypes.byref(_kv(**bad)))).values())
    assert rc < 0 and text in L.qlin_last_error().decode(), L.qlin_last_error()


def test_shared_empty_calls(S):
    L = _lib(S)
    for none in (dict(B=0), dict(G=0)):
        assert L.qlin_attn_decode_shared(*(SHARED | dict(kv=ctypes.byref(_kv()), q=None, out=None, ws=None) | none).values()) == 0


LOGITS = dict(logits=FAKE, logits_row=1000, out=2 * FAKE, out_row=1000, tokens=3 * FAKE, tokens_row=50, lens=4 * FAKE,
              prompt_lens=4 * FAKE + 64, bias_ids=5 * FAKE, bias_ids_row=9, bias=6 * FAKE, bias_row=9, mask=7 * FAKE,
              mask_row=32, B=2, V=1000, history=50, biases=9, dtype=2, out_dtype=3, repetition_all=1.0)


@pytest.mark.parametrize("bad,text", [
    (dict(B=-1), "negative"), (dict(V=-1), "negative"), (dict(history=-1), "negative"), (dict(biases=-1), "negative"),
    (dict(B=(1 << 16) + 1), "more than 65536 rows"), (dict(V=(1 << 30) + 1), "vocabulary"), (dict(history=(1 << 30) + 1), "more than"),
    (dict(dtype=4), "logits of dtype"), (dict(out_dtype=0), "out of dtype"), (dict(logits=None), "null logits"),
    (dict(out=None), "null out"), (dict(tokens=None), "null tokens"), (dict(bias=None), "null bias"),
    (dict(bias_ids=None), "null bias_ids"), (dict(logits=FAKE + 1), "logits must be 2-byte"), (dict(out=2 * FAKE + 2), "out must be 4-byte"),
    (dict(tokens=3 * FAKE + 4, tokens_64=1), "tokens must be 8-byte"), (dict(lens=FAKE + 2), "lengths must be 4-byte"),
    (dict(mask=7 * FAKE + 2), "mask must be 4-byte"), (dict(out_row=999), "rows of out overlap"), (dict(logits_row=-1), "overlap"),
    (dict(repetition_all=0.0), "repetition must be"), (dict(repetition_all=float("nan")), "repetition must be"),
    (dict(presence_all=float("inf")), "presence must be"), (dict(frequency_all=float("nan")), "frequency must be"),
    (dict(repetition=FAKE + 2), "repetition must be 4-byte"), (dict(out=FAKE + 4), "out overlaps logits"),
    (dict(out=FAKE), "out overlaps logits"), (dict(out=3 * FAKE + 32), "out overlaps tokens"),
    (dict(out=4 * FAKE - 4000), "out overlaps lens"), (dict(out=5 * FAKE), "out overlaps bias_ids"),
    (dict(out=6 * FAKE), "out overlaps bias"), (dict(out=7 * FAKE), "out overlaps mask"),
    (dict(mask_bytes=1, mask=2 * FAKE - 1), "out overlaps mask"), (dict(presence=2 * FAKE), "out overlaps presence"),
    (dict(B=1 << 16, V=1 << 20, logits_row=1 << 20, out_row=1 << 20, out=1 << 46, logits=1 << 45), "too many logits"),
])
def test_logits_refusals(S, bad, text):
    L = _lib(S)
    rc = L.qlin_logits_process(ctypes.byref(Logits(**(LOGITS | bad))), None)
    assert rc < 0 and text in L.qlin_last_error().decode(), L.qlin_last_error()
    assert L.qlin_logits_process(None, None) < 0


def test_logits_empty_calls(S):
    L = _lib(S)
    for none in (dict(B=0), dict(V=0)):
        assert L.qlin_logits_process(ctypes.byref(Logits(**(LOGITS | dict(logits=None, out=None) | none))), None) == 0


SAMPLE = dict(logits=FAKE, dt=3, row=1000, B=2, V=1000, k=20, u=2 * FAKE, t=None, ta=1.0, p=None, pa=1.0, m=None, ma=0.0,
              tokens=3 * FAKE, t64=1, lp=4 * FAKE, ws=8 * FAKE, nws=256 << 20, st=None)


@pytest.mark.parametrize("bad,text", [
    (dict(B=-1), "negative"), (dict(V=-1), "negative"), (dict(V=0), "empty vocabulary"), (dict(B=(1 << 16) + 1), "more than 65536 rows"),
    (dict(V=(1 << 30) + 1), "vocabulary"), (dict(dt=7), "dtype"), (dict(k=0), "top_k"), (dict(k=129), "top_k"), (dict(k=-3), "top_k"),
    (dict(ta=-0.5), "temperature"), (dict(ta=float("nan")), "temperature"), (dict(ta=float("inf")), "temperature"),
    (dict(pa=-1.0), "top_p"), (dict(pa=float("nan")), "top_p"), (dict(ma=-0.1), "min_p"), (dict(logits=None), "null logits"),
    (dict(u=None), "null u"), (dict(tokens=None), "null tokens"), (dict(u=FAKE + 2), "u must be 4-byte"),
    (dict(tokens=3 * FAKE + 4), "tokens must be 8-byte"), (dict(lp=FAKE + 2), "logprobs must be 4-byte"),
    (dict(t=FAKE + 1), "temperature must be 4-byte"), (dict(row=-5), "overlap"), (dict(tokens=2 * FAKE), "tokens overlaps u"),
    (dict(lp=2 * FAKE), "logprobs overlaps u"), (dict(tokens=FAKE + 800), "tokens overlaps logits"), (dict(lp=3 * FAKE), "overlaps logprobs"),
    (dict(p=4 * FAKE), "logprobs overlaps top_p"), (dict(ws=None), "workspace"), (dict(nws=5 << 20), "workspace too small"),
    (dict(ws=8 * FAKE + 16), "256-byte"),
])
def test_sample_refusals(S, bad, text):
    L = _lib(S)
    rc = L.qlin_sample(*(SAMPLE | bad).values())
    assert rc < 0 and text in L.qlin_last_error().decode(), L.qlin_last_error()


def test_sample_empty_call(S):
    L = _lib(S)
    assert L.qlin_sample(*(SAMPLE | dict(B=0, logits=None, u=None, tokens=None, ws=None)).values()) == 0


# ------------------------------------------------------------------ the Python calls

def test_shared_python_checks():
    from qwen35_amd.kernels import attention as A
    q = torch.zeros((3, 8, 64), dtype=BF)
    kc = torch.zeros((4, 16, 2, 64), dtype=BF)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    good = dict(q=q, k=kc, v=kc.clone(), pt=i(2, 3), pl=i(2), cu=i(3), t=i(3, 2), n=i(3), out=q.clone())

    def call(**bad):
        a = good | bad
        return A.attn_decode_shared(a["q"], a["k"], a["v"], a["pt"], a["pl"], a["cu"], a["t"], a["n"], a["out"])

    for bad, text in ((dict(), "GPU"), (dict(q=q.float()), "bfloat16 or float16"), (dict(pt=i(1, 3)), "prefix_table must be"),
                      (dict(pt=i(2, 3).long()), "prefix_table must be int32"), (dict(pl=i(3)), "prefix_len must be"),
                      (dict(cu=i(2, 2)), "cu_seq must be"), (dict(cu=i(0)), "cu_seq must be"), (dict(cu=i(3).long()), "cu_seq must be"),
                      (dict(t=i(2, 2)), "table must be"), (dict(n=i(2)), "kv_len must be"), (dict(out=q[:2]), "out must have"),
                      (dict(k=kc[..., :32]), "must both be")):
        with pytest.raises(ValueError, match=text):
            call(**bad)


def test_logits_python_checks(S):
    x = torch.zeros((2, 40))
    t = torch.zeros((2, 5), dtype=torch.int32)
    w = torch.zeros((2, 2), dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    for kw, text in (
            (dict(), "GPU"), (dict(logits=x.double()), "bfloat16, float16 or float32"), (dict(out=x.double()), "out must be"),
            (dict(out=x[:1]), "out must be"), (dict(logits=x[0]), "logits must be"), (dict(logits=x.t()), "contiguous"),
            (dict(tokens=t[:1]), "tokens must be"), (dict(tokens=t.float()), "tokens must be"), (dict(lens=n), "need tokens"),
            (dict(repetition=1.1), "need tokens"), (dict(presence=torch.zeros(2)), "need tokens"),
            (dict(tokens=t, lens=n.long()), "lens must be"), (dict(tokens=t, prompt_lens=n[:1]), "prompt_lens must be"),
            (dict(tokens=t, repetition=torch.ones(3)), "repetition must be"), (dict(tokens=t, frequency=torch.ones(2).double()), "frequency must be"),
            (dict(bias=x[:, :5]), "take bias_ids"), (dict(bias_ids=t), "take bias_ids"), (dict(bias_ids=t, bias=x[:, :4]), "bias must be"),
            (dict(bias_ids=t.long(), bias=x[:, :5]), "bias_ids must be"), (dict(mask=w[:, :1]), "mask must be"),
            (dict(mask=x > 0), "GPU"), (dict(mask=(x > 0)[:, :39]), "mask must be"), (dict(mask=w.long()), "mask must be")):
        a = dict(logits=x, out=x.clone()) | kw
        with pytest.raises(ValueError, match=text):
            S.logits_process(a.pop("logits"), a.pop("out"), **a)


def test_sample_python_checks(S):
    x, u, tok = torch.zeros((2, 40)), torch.zeros(2), torch.zeros(2, dtype=torch.int64)
    for kw, text in (
            (dict(), "GPU"), (dict(logits=x.int()), "logits must be"), (dict(u=u[:1]), "u must be"), (dict(u=u.double()), "u must be"),
            (dict(tokens=tok.float()), "tokens must be"), (dict(tokens=tok[:1]), "tokens must be"), (dict(logprobs=u.double()), "logprobs must be"),
            (dict(temperature=torch.ones(1)), "temperature must be"), (dict(top_p=u.double()), "top_p must be"),
            (dict(min_p=torch.zeros((2, 1))), "min_p must be"), (dict(u=torch.zeros((2, 2))[:, 0]), "contiguous")):
        a = dict(logits=x, u=u, tokens=tok) | kw
        with pytest.raises(ValueError, match=text):
            S.sample(a.pop("logits"), a.pop("u"), a.pop("tokens"), **a)
