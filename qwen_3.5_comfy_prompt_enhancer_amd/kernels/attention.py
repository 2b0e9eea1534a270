"""What an attention layer does between its projections and its output projection.

The reference's kernels/attention.py holds these steps as qk_norm_rope (111-134),
attn_prefill (196-206) and attn_decode (256-267) over a cache of its own; here they read
and write a paged cache, which several sequences share and a page table orders:

* `qk_norm_rope`       RMSNorm of every query and key head, rotary positions of one to
                       three axes, keys and values into the cache;
* `attn_prompt`        attention of packed prompts over their own keys;
* `attn_prompt_paged`  attention of the next chunk of prompts over the cache;
* `attn_decode`        attention of one new token of each sequence over the cache.

A step of an attention layer, from proj3's rows to the output projection's producer:

    qk_norm_rope(proj[:, :2 * HQ * HD].view(T, HQ, 2 * HD)[..., :HD], k, pos, freqs, q, v=v,
                 k_cache=kc, v_cache=vc, slots=slots, q_w=wq, k_w=wk)
    attn_decode(q, kc, vc, table, kv_len, out)               # or attn_prompt_paged
    gate_mul_quant(out.view(T, HQ * HD), proj[:, :2 * HQ * HD], aq, a_s, hd=HD)

Cache tensors are [pages, page, kv_heads, hd] (a power of two tokens to a page, 16 to
1024) with any strides in front of the last axis, so a buffer that is laid out
[pages, kv_heads, page, hd] passes as its permuted view.  They hold the queries' type, or
int8 codes with fp32 scales k_s / v_s [pages, page, kv_heads].  16-bit tensors need
16-byte aligned rows (strides that are multiples of 8; int8: of 16).

Lengths, page tables, slots and positions stay on the device and are never waited for;
what they may hold is stated in include/qlin_attn.h.  All calls run on the current
stream of their tensors' device and can be captured (see `qlin.capture`).
"""
from __future__ import annotations

import ctypes

import torch

from . import qlin as C

__all__ = ["qk_norm_rope", "attn_prompt", "attn_prompt_paged", "attn_decode"]

QLIN_I8 = 4

_P, _I, _L, _S, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float


class _PagedKV(ctypes.Structure):
    """include/qlin_attn.h qlin_paged_kv."""
    _fields_ = [
        ("k", _P), ("k_page", _L), ("k_token", _L), ("k_head", _L),
        ("v", _P), ("v_page", _L), ("v_token", _L), ("v_head", _L),
        ("k_s", _P), ("ks_page", _L), ("ks_token", _L), ("ks_head", _L),
        ("v_s", _P), ("vs_page", _L), ("vs_token", _L), ("vs_head", _L),
        ("dtype", _I), ("num_pages", _I), ("page", _I),
    ]


class _Rope(ctypes.Structure):
    """include/qlin_attn.h qlin_rope."""
    _fields_ = [
        ("q", _P), ("q_token", _L), ("q_head", _L),
        ("k", _P), ("k_token", _L), ("k_head", _L),
        ("v", _P), ("v_token", _L), ("v_head", _L),
        ("q_out", _P), ("qo_token", _L), ("qo_head", _L),
        ("k_out", _P), ("ko_token", _L), ("ko_head", _L),
        ("cache", ctypes.POINTER(_PagedKV)), ("slots", _P), ("slots_64", _I),
        ("pos", _P), ("pos_axis", _L), ("pos_token", _L), ("pos_64", _I),
        ("freqs", _P), ("freqs_64", _I),
        ("q_w", _P), ("k_w", _P), ("w_dtype", _I), ("one_plus", _I), ("eps", _F),
        ("T", _I), ("q_heads", _I), ("kv_heads", _I), ("hd", _I), ("rot", _I), ("axes", _I),
        ("sections", _I * 3), ("interleaved", _I), ("dtype", _I),
    ]


_KV = ctypes.POINTER(_PagedKV)
_SIGS = {
    "qlin_qk_norm_rope": [ctypes.POINTER(_Rope), _P],
    "qlin_attn_prompt": [_P, _L, _L, _P, _L, _L, _P, _L, _L, _P, _P, _P, _L, _L, _I, _I, _I, _I, _I, _I, _I, _F, _I,
                         _P, _S, _P],
    "qlin_attn_prompt_paged": [_P, _L, _L, _KV, _P, _L, _I, _P, _P, _P, _L, _L, _I, _I, _I, _I, _I, _I, _F, _I,
                               _P, _S, _P],
    "qlin_attn_decode": [_P, _L, _L, _KV, _P, _L, _I, _P, _P, _L, _L, _I, _I, _I, _I, _I, _F, _P, _S, _P],
}
EXPORTS = tuple(_SIGS)

_fns: dict = {}


def _call(name, device, *args):
    """One C entry point on `device`, which need not be the current one."""
    f = _fns.get(name)
    if f is None:
        f = getattr(C.lib(), name)
        f.restype = ctypes.c_int
        f.argtypes = _SIGS[name]
        _fns[name] = f
    if torch.cuda.current_device() == device:
        status = f(*args)
    else:
        with torch.cuda.device(device):
            status = f(*args)
    if status != C.QLIN_OK:
        C.check(status, name)


def _rows(name, t, heads, hd, dtype):
    """A [rows, heads, hd] tensor of 16-bit values with a contiguous last axis."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != hd:
        raise ValueError(f"{name} must be [rows, {heads}, {hd}], not {list(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    if t.stride(2) != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")


def _queries(q):
    if q.dim() != 3:
        raise ValueError("q must be [rows, heads, hd]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("q must be bfloat16 or float16")
    if q.stride(2) != 1:
        raise ValueError("the last axis of q must be contiguous")
    return q.shape


def _ints(name, t, shape=None, dtypes=(torch.int32,)):
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")


def _cache(k, v, k_s, v_s, dtype, hd):
    """The C view of a cache, and its key heads."""
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError("k_cache and v_cache must both be [pages, page, kv_heads, hd]")
    pages, page, heads, d = k.shape
    if d != hd:
        raise ValueError(f"the cache's head size {d} is not the queries' {hd}")
    if k.dtype != v.dtype:
        raise ValueError("k_cache and v_cache must share a dtype")
    if k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError("the last axis of the cache must be contiguous")
    if k.dtype == torch.int8:
        if k_s is None or v_s is None:
            raise ValueError("an int8 cache needs its scales k_s and v_s")
        for name, s in (("k_s", k_s), ("v_s", v_s)):
            if s.dtype != torch.float32 or s.shape != k.shape[:3]:
                raise ValueError(f"{name} must be float32 {[pages, page, heads]}")
        return _PagedKV(k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], k_s.data_ptr(), *k_s.stride(),
                        v_s.data_ptr(), *v_s.stride(), QLIN_I8, pages, page), heads
    if k.dtype != dtype:
        raise ValueError(f"the cache must be int8 or {dtype}")
    if k_s is not None or v_s is not None:
        raise ValueError("a 16-bit cache has no scales")
    return _PagedKV(k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], None, 0, 0, 0, None, 0, 0, 0,
                    C.dtype_code(k), pages, page), heads


def qk_norm_rope(q, k, pos, freqs, q_out, k_out=None, v=None, k_cache=None, v_cache=None, slots=None, k_s=None,
                 v_s=None, q_w=None, k_w=None, eps=1e-6, one_plus=True, sections=None, interleaved=False):
    """RMSNorm and rotary positions of queries and keys; keys and values into the cache.

    q [T, q_heads, hd], k [T, kv_heads, hd] (views of a projection's rows will do).
    With q_w / k_w [hd], each head becomes `x * rsqrt(mean(x^2) + eps) * (w + 1 if
    one_plus else w)`; then the pairs (i, i + r/2) of its first r = 2 * len(freqs) values
    (a multiple of 16) turn by `pos[axis(i)] * freqs[i]`, an angle taken in 64 bits.
    pos: int32 or int64 [T] or [axes, T]; freqs: float32 or float64 [r/2].  `sections`
    gives the frequencies of each axis: consecutive runs, or with `interleaved` axes in
    turn (frequency i to axis i % axes while that axis has frequencies left, then to axis
    0); default: all to the first axis, which several axes do not have.

    q_out [T, q_heads, hd] and k_out [T, kv_heads, hd] (optional with a cache) may be q
    and k themselves.  With k_cache / v_cache, token t's key and v [T, kv_heads, hd] go to
    slot slots[t] = page * page_size + place (int32 or int64; a negative slot, or one past
    the cache, stores nothing; a slot given twice holds one of the two, whole or mixed by
    head).  An int8 cache gets codes round_half_away(y / s) with `s = max(amax / 127,
    1e-8)` of each token's head in k_s / v_s.  Returns q_out."""
    T, hq, hd = _queries(q)
    dt = q.dtype
    if k.dim() != 3:
        raise ValueError("k must be [rows, kv_heads, hd]")
    hkv = k.shape[1]
    _rows("k", k, hkv, hd, dt)
    _rows("q_out", q_out, hq, hd, dt)
    if k.shape[0] != T or q_out.shape[0] != T:
        raise ValueError(f"q, k and q_out must have the same rows ({T})")
    if pos.dim() == 1:
        pos = pos[None]
    if pos.dim() != 2 or pos.shape[1] != T:
        raise ValueError(f"pos must be [{T}] or [axes, {T}]")
    if pos.dtype not in (torch.int32, torch.int64):
        raise ValueError("pos must be int32 or int64")
    if freqs.dim() != 1 or freqs.dtype not in (torch.float32, torch.float64) or not freqs.is_contiguous():
        raise ValueError("freqs must be a contiguous float32 or float64 vector")
    half, axes = freqs.shape[0], pos.shape[0]
    if sections is None:
        if axes != 1:
            raise ValueError(f"{axes} position axes need sections")
        sections = (half,)
    if len(sections) != axes:
        raise ValueError(f"sections must give one length for each of the {axes} axes")
    if axes > 3:
        raise ValueError("at most 3 position axes")
    for name, w in (("q_w", q_w), ("k_w", k_w)):
        if w is not None and (w.dim() != 1 or w.shape[0] != hd or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous [{hd}]")
    if q_w is not None and k_w is not None and q_w.dtype != k_w.dtype:
        raise ValueError("q_w and k_w must share a dtype")
    w = q_w if q_w is not None else k_w
    if k_out is not None:
        _rows("k_out", k_out, hkv, hd, dt)
        if k_out.shape[0] != T:
            raise ValueError(f"k_out must have {T} rows")
    cache = None
    if k_cache is not None or v_cache is not None or slots is not None:
        if k_cache is None or v_cache is None or v is None or slots is None:
            raise ValueError("a cache takes k_cache, v_cache, v and slots")
        _rows("v", v, hkv, hd, dt)
        _ints("slots", slots, (T,), (torch.int32, torch.int64))
        if v.shape[0] != T:
            raise ValueError(f"v must have {T} rows")
        cache, ch = _cache(k_cache, v_cache, k_s, v_s, dt, hd)
        if ch != hkv:
            raise ValueError(f"the cache has {ch} key heads, k {hkv}")
    elif k_out is None:
        raise ValueError("give k_out, a cache, or both")
    C.require_cuda(q, k, v, pos, freqs, q_out, k_out, k_cache, v_cache, slots, k_s, v_s, q_w, k_w)
    dev = q.get_device()
    args = _Rope(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
        C.ptr(v), v.stride(0) if v is not None else 0, v.stride(1) if v is not None else 0,
        q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
        C.ptr(k_out), k_out.stride(0) if k_out is not None else 0, k_out.stride(1) if k_out is not None else 0,
        ctypes.pointer(cache) if cache is not None else None, C.ptr(slots),
        1 if slots is not None and slots.dtype == torch.int64 else 0,
        pos.data_ptr(), pos.stride(0), pos.stride(1), 1 if pos.dtype == torch.int64 else 0,
        freqs.data_ptr(), 1 if freqs.dtype == torch.float64 else 0,
        C.ptr(q_w), C.ptr(k_w), C.dtype_code(w) if w is not None else 0, 1 if one_plus else 0, float(eps),
        T, hq, hkv, hd, 2 * half, axes, (_I * 3)(*sections), 1 if interleaved else 0, C.dtype_code(q))
    _call("qlin_qk_norm_rope", dev, ctypes.byref(args), C.current_stream(dev))
    return q_out


def attn_prompt(q, k, v, cu_q, out, cu_k=None, scale=None, causal=True):
    """Attention of packed prompts: sequence b's queries are rows cu_q[b] .. cu_q[b + 1] - 1
    of q [T, q_heads, hd], its keys and values rows cu_k[b] .. (default: cu_q) of k, v
    [Tk, kv_heads, hd].  cu_q, cu_k: int32 [B + 1], rising from 0.  `causal`: query i of a
    sequence sees its keys j <= i + keys - queries (the last query sees all).  scale:
    hd ** -0.5 unless given.  out [T, q_heads, hd]; a row that sees no key is zero, rows of
    no sequence stay as they were.  Returns out."""
    T, hq, hd = _queries(q)
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError("k and v must both be [rows, kv_heads, hd]")
    hkv = k.shape[1]
    _rows("k", k, hkv, hd, q.dtype)
    _rows("v", v, hkv, hd, q.dtype)
    _rows("out", out, hq, hd, q.dtype)
    if out.shape[0] != T:
        raise ValueError(f"out must have {T} rows")
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must be [sequences + 1]")
    _ints("cu_q", cu_q)
    if cu_k is None:
        if k.shape[0] != T:
            raise ValueError("k and v must have the queries' rows, or cu_k be given")
        cu_k = cu_q
    _ints("cu_k", cu_k, tuple(cu_q.shape))
    C.require_cuda(q, k, v, cu_q, cu_k, out)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_prompt", out.get_device(), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
          k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(),
          out.stride(0), out.stride(1), T, k.shape[0], cu_q.shape[0] - 1, hq, hkv, hd, C.dtype_code(q),
          hd ** -0.5 if scale is None else float(scale), 1 if causal else 0, ws, nws, stream)
    return out


def attn_prompt_paged(q, k_cache, v_cache, table, kv_len, cu_q, out, k_s=None, v_s=None, scale=None, causal=True):
    """`attn_prompt` over the cache, for a chunk of each prompt: sequence b's keys are the
    first kv_len[b] tokens of pages table[b, 0], table[b, 1], ... (its chunk's own among
    them: store them first).  table: int32 [B, pages a sequence], kv_len: int32 [B], cu_q:
    int32 [B + 1].  Returns out."""
    T, hq, hd = _queries(q)
    cache, hkv = _cache(k_cache, v_cache, k_s, v_s, q.dtype, hd)
    _rows("out", out, hq, hd, q.dtype)
    if out.shape[0] != T:
        raise ValueError(f"out must have {T} rows")
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must be [sequences + 1]")
    B = cu_q.shape[0] - 1
    _ints("cu_q", cu_q)
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table must be [{B}, pages]")
    _ints("table", table)
    _ints("kv_len", kv_len, (B,))
    C.require_cuda(q, k_cache, v_cache, table, kv_len, cu_q, out, k_s, v_s)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_prompt_paged", out.get_device(), q.data_ptr(), q.stride(0), q.stride(1), ctypes.byref(cache),
          table.data_ptr(), table.stride(0), table.shape[1], kv_len.data_ptr(), cu_q.data_ptr(), out.data_ptr(),
          out.stride(0), out.stride(1), T, B, hq, hkv, hd, C.dtype_code(q),
          hd ** -0.5 if scale is None else float(scale), 1 if causal else 0, ws, nws, stream)
    return out


def attn_decode(q, k_cache, v_cache, table, kv_len, out, k_s=None, v_s=None, scale=None):
    """Attention of one new token of each sequence: q and out [B, q_heads, hd]; sequence b's
    keys are the first kv_len[b] tokens (the new one among them) of pages table[b, 0],
    table[b, 1], ...  table: int32 [B, pages a sequence], kv_len: int32 [B].  A sequence
    without keys gives zeros.  scale: hd ** -0.5 unless given.  Returns out."""
    B, hq, hd = _queries(q)
    cache, hkv = _cache(k_cache, v_cache, k_s, v_s, q.dtype, hd)
    _rows("out", out, hq, hd, q.dtype)
    if out.shape[0] != B:
        raise ValueError(f"out must have {B} rows")
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table must be [{B}, pages]")
    _ints("table", table)
    _ints("kv_len", kv_len, (B,))
    C.require_cuda(q, k_cache, v_cache, table, kv_len, out, k_s, v_s)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_decode", out.get_device(), q.data_ptr(), q.stride(0), q.stride(1), ctypes.byref(cache),
          table.data_ptr(), table.stride(0), table.shape[1], kv_len.data_ptr(), out.data_ptr(), out.stride(0),
          out.stride(1), B, hq, hkv, hd, C.dtype_code(q), hd ** -0.5 if scale is None else float(scale), ws, nws,
          stream)
    return out
