"""Runs calls of the attention operators' C ABI on the CPU over the recording HIP runtime of fake_hip.cpp
and returns what each would have launched (as dispatch.py does for the linears; these calls have
structs and floats).  Device pointers are invented addresses, far apart unless a test moves them."""
from __future__ import annotations

import ctypes
import json
import pathlib
import subprocess
import sys

TESTS = pathlib.Path(__file__).resolve().parent
LIB = TESTS.parent / "qwen_3.5_comfy_prompt_enhancer_amd" / "kernels" / "libqlin.so"
BF16, F16, I8 = 2, 1, 4
Q, K, V, OUT, KO, TABLE, LEN, CU, WS, KS, VS, POS, FREQS, W, SLOTS = ((i + 1) << 44 for i in range(15))


class PagedKV(ctypes.Structure):
    """include/qlin_attn.h qlin_paged_kv."""
    _fields_ = [(f, t) for x in ("k", "v", "k_s", "v_s")
                for f, t in ((x, ctypes.c_void_p), *((x.replace("_", "") + s, ctypes.c_int64)
                                                     for s in ("_page", "_token", "_head")))]
    _fields_ += [(f, ctypes.c_int) for f in ("dtype", "num_pages", "page")]


class Rope(ctypes.Structure):
    """include/qlin_attn.h qlin_rope."""
    _fields_ = [(f, {"p": ctypes.c_void_p, "l": ctypes.c_int64, "i": ctypes.c_int, "f": ctypes.c_float}[t])
                for t, f in (x.split(":") for x in (
                    "p:q l:q_token l:q_head p:k l:k_token l:k_head p:v l:v_token l:v_head p:q_out l:qo_token "
                    "l:qo_head p:k_out l:ko_token l:ko_head p:slots i:slots_64 p:pos l:pos_axis l:pos_token "
                    "i:pos_64 p:freqs i:freqs_64 p:q_w p:k_w i:w_dtype i:one_plus f:eps i:T i:q_heads i:kv_heads "
                    "i:hd i:rot i:axes i:s0 i:s1 i:s2 i:interleaved i:dtype").split())]


def cache(heads, hd, pages=8, page=64, dtype=BF16, **kw):
    """A cache [pages][page][heads][hd]."""
    d = dict(k=K, k_page=page * heads * hd, k_token=heads * hd, k_head=hd, v=V, v_page=page * heads * hd,
             v_token=heads * hd, v_head=hd, dtype=dtype, num_pages=pages, page=page)
    if dtype == I8:
        d |= dict(k_s=KS, ks_page=page * heads, ks_token=heads, ks_head=1, v_s=VS, vs_page=page * heads,
                  vs_token=heads, vs_head=1)
    return d | kw


def decode(kv, B=2, hq=8, hkv=4, hd=64, table=TABLE, max_pages=8, dt=BF16, **kw):
    d = dict(q=Q, qs=hq * hd, qh=hd, kv=kv, table=table, ts=max_pages, mp=max_pages, kv_len=LEN, out=OUT, os=hq * hd,
             oh=hd, B=B, hq=hq, hkv=hkv, hd=hd, dt=dt, scale=0.125, ws=WS, nws=256 << 20, st=None)
    return ["qlin_attn_decode", *(d | kw).values()]


def paged(kv, T=9, B=2, hq=8, hkv=4, hd=64, table=TABLE, max_pages=8, dt=BF16, **kw):
    d = dict(q=Q, qt=hq * hd, qh=hd, kv=kv, table=table, ts=max_pages, mp=max_pages, kv_len=LEN, cu=CU, out=OUT,
             ot=hq * hd, oh=hd, T=T, B=B, hq=hq, hkv=hkv, hd=hd, dt=dt, scale=0.125, causal=1, ws=WS, nws=256 << 20,
             st=None)
    return ["qlin_attn_prompt_paged", *(d | kw).values()]


def prompt(T=9, Tk=None, B=2, hq=8, hkv=4, hd=64, dt=BF16, **kw):
    d = dict(q=Q, qt=hq * hd, qh=hd, k=K, kt=hkv * hd, kh=hd, v=V, vt=hkv * hd, vh=hd, cu=CU, ck=CU, out=OUT, ot=hq * hd,
             oh=hd, T=T, Tk=T if Tk is None else Tk, B=B, hq=hq, hkv=hkv, hd=hd, dt=dt, scale=0.125, causal=1, ws=WS,
             nws=256 << 20, st=None)
    return ["qlin_attn_prompt", *(d | kw).values()]


def rope(kv=None, T=4, hq=8, hkv=4, hd=64, **kw):
    d = dict(q=Q, q_token=hq * hd, q_head=hd, k=K, k_token=hkv * hd, k_head=hd, v=V + (1 << 43), v_token=hkv * hd,
             v_head=hd, q_out=OUT, qo_token=hq * hd, qo_head=hd, k_out=KO, ko_token=hkv * hd, ko_head=hd, slots=SLOTS,
             pos=POS, pos_axis=T, pos_token=1, freqs=FREQS, q_w=W, k_w=W, w_dtype=2, one_plus=1, eps=1e-6, T=T,
             q_heads=hq, kv_heads=hkv, hd=hd, rot=64, axes=1, s0=32, s1=0, s2=0, interleaved=0, dtype=BF16)
    if kv is not None and "k" not in kw:
        d["k"] = K + (1 << 43)
    return ["qlin_qk_norm_rope", {"rope": d | kw}, kv, None]


def run(tmp, calls):
    """[(status, [kernel name, grid x, ...], message)] of each call."""
    fake = pathlib.Path(tmp) / "libfake_hip.so"
    if not fake.exists():
        subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", str(fake), str(TESTS / "fake_hip.cpp")], check=True)
    r = subprocess.run([sys.executable, __file__, str(fake), str(LIB)], input=json.dumps(calls), text=True,
                       capture_output=True)
    assert r.returncode == 0, r.stderr
    return [(st, [(k, g) for k, g in ev], msg) for st, ev, msg in json.loads(r.stdout)]


def _child(fake, lib):
    f = ctypes.CDLL(fake, mode=ctypes.RTLD_GLOBAL)
    f.fake_log.restype = ctypes.c_char_p
    q = ctypes.CDLL(lib)
    q.qlin_last_error.restype = ctypes.c_char_p

    def arg(a):
        if isinstance(a, dict):
            return ctypes.byref(Rope(**a["rope"]) if "rope" in a else PagedKV(**a))
        return None if a is None else ctypes.c_float(a) if isinstance(a, float) else ctypes.c_int64(a)

    out = []
    for name, *args in json.load(sys.stdin):
        f.fake_clear()
        status = getattr(q, name)(*map(arg, args))
        log = [line.split() for line in f.fake_log().decode().splitlines()]
        out.append((status, [(x[1], int(x[2])) for x in log if x[0] == "launch"], q.qlin_last_error().decode()))
    json.dump(out, sys.stdout)


if __name__ == "__main__":
    _child(*sys.argv[1:])
