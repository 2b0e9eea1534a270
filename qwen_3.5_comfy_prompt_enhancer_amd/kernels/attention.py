"""What an attention layer does between its projections and its output projection.

The reference's kernels/attention.py holds these steps as qk_norm_rope (111-134),
attn_prefill (196-206) and attn_decode (256-267) over a cache of its own; here they read
and write a paged cache, which several sequences share and a page table orders:

* `qk_norm_rope`       RMSNorm of every query and key head, rotary positions of one to
                       three axes, keys and values into the cache;
* `attn_prompt`        attention of packed prompts over their own keys;
* `attn_prompt_paged`  attention of the next chunk of prompts over the cache;
* `attn_decode`        attention of one new token of each sequence over the cache;
* `attn_decode_shared` the same for groups of sequences that share a prefix, whose keys are
                       read once for the group.

A step of an attention layer, from proj3's rows to the output projection's producer:

    qk_norm_rope(proj[:, :2 * HQ * HD].view(T, HQ, 2 * HD)[..., :HD], k, pos, freqs, q, v=v,
                 k_cache=kc, v_cache=vc, slots=slots, q_w=wq, k_w=wk)
    attn_decode(q, kc, vc, table, kv_len, out)               # or attn_prompt_paged
    gate_mul_quant(out.view(T, HQ * HD), proj[:, :2 * HQ * HD], aq, a_s, hd=HD)

Cache tensors are [pages, page, kv_heads, hd] (a power of two tokens to a page, 16 to
1024) with any strides in front of the last axis, so a buffer that is laid out
[pages, kv_heads, page, hd] passes as its permuted view.  They hold the queries' type, or
int8 codes with fp32 scales k_s / v_s [pages, page, kv_heads].  16-bit tensors need
16-byte aligned rows (strides that are multiples of 8; int8: of 16; of tokens at most 2^26
elements, of heads and pages 2^31 - 16).

What a call writes shares no memory with what it reads (`qk_norm_rope` in place aside): such calls are
refused.  Lengths, page tables, slots and positions stay on the device and are never waited for;
what they may hold is stated in include/qlin_attn.h.  All calls run on the current
stream of their tensors' device and can be captured (see `qlin.capture`).
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import qlin as C

__all__ = ["qk_norm_rope", "attn_prompt", "attn_prompt_paged", "attn_decode", "attn_decode_shared"]

QLIN_I8 = 4

_P, _I, _L, _S, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
_B = ctypes.c_char_p  # a struct of the ABI, packed (a third of the time of a ctypes.Structure)

# include/qlin_attn.h qlin_paged_kv: four times a pointer and three strides; dtype, pages, page size
_PAGED_KV = struct.Struct("@" + 4 * "P3q" + "3i0q")
# qlin_rope: q, k, v, q_out, k_out with two strides; slots; positions; frequencies; norm;
# sizes
_ROPE = struct.Struct("@" + 5 * "P2q" + "Pi" + "P2qi" + "Pi" + "PP2if" + "6i" + "3i" + "2i0q")

_SIGS = {
    "qlin_qk_norm_rope": [_B, _B, _P],
    "qlin_attn_prompt": [_P, _L, _L, _P, _L, _L, _P, _L, _L, _P, _P, _P, _L, _L, _I, _I, _I, _I, _I, _I, _I, _F, _I,
                         _P, _S, _P],
    "qlin_attn_prompt_paged": [_P, _L, _L, _B, _P, _L, _I, _P, _P, _P, _L, _L, _I, _I, _I, _I, _I, _I, _F, _I,
                               _P, _S, _P],
    "qlin_attn_decode": [_P, _L, _L, _B, _P, _L, _I, _P, _P, _L, _L, _I, _I, _I, _I, _I, _F, _P, _S, _P],
}
EXPORTS = tuple(_SIGS)  # of include/qlin_attn.h
# include/qlin_candidates.h
_SIGS["qlin_attn_decode_shared"] = [_P, _L, _L, _B, _P, _L, _I, _P, _P, _I, _P, _L, _I, _P, _P, _L, _L, _I, _I, _I,
                                    _I, _I, _F, _P, _S, _P]

_DT = {torch.bfloat16: C.QLIN_BF16, torch.float16: C.QLIN_F16}
_WDT = {**_DT, torch.float32: C.QLIN_F32}
_INTS = (torch.int32, torch.int64)
_fns: dict = {}
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(name, device, *args):
    """One C entry point on `device`, which need not be the current one."""
    f = _fns.get(name)
    if f is None:
        f = getattr(C.lib(), name)
        f.restype = ctypes.c_int
        f.argtypes = _SIGS[name]
        _fns[name] = f
    if _current_device() == device:
        status = f(*args)
    else:
        with torch.cuda.device(device):
            status = f(*args)
    if status != C.QLIN_OK:
        C.check(status, name)


_INT_MAX = (1 << 31) - 1  # of the ABI's sizes: a ctypes int keeps 32 bits of a larger one


def _size(name, n):
    if n > _INT_MAX:
        raise ValueError(f"{name}: {n} is more than {_INT_MAX}")
    return n


def _strides(name, t, rows, heads, hd, dtype):
    """Row and head strides of a [rows, heads, hd] tensor of 16-bit values whose last axis is
    contiguous."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != hd:
        raise ValueError(f"{name} must be [rows, {heads}, {hd}], not {list(shape)}")
    if shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    st = t.stride()
    if st[2] != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")
    return st[0], st[1]


def _queries(q):
    """Rows, heads, head size, type code and strides of the queries."""
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q must be [rows, heads, hd]")
    dt = _DT.get(q.dtype)
    if dt is None:
        raise ValueError("q must be bfloat16 or float16")
    st = q.stride()
    if st[2] != 1:
        raise ValueError("the last axis of q must be contiguous")
    if shape[0] > _INT_MAX or shape[1] > _INT_MAX:
        _size("rows and heads of q", max(shape))
    return *shape, dt, st[0], st[1]


def _vector(name, t, n, dtypes=(torch.int32,)):
    if t.dtype in dtypes and t.dim() == 1 and t.numel() == n and t.is_contiguous():
        return  # (half the time of reading its shape and strides)
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}")
    shape = t.shape
    if len(shape) != 1 or shape[0] != n:
        raise ValueError(f"{name} must be [{n}], not {list(shape)}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")


def _weight(name, w, hd):
    """Type code of a norm's weights."""
    shape, dt = w.shape, _WDT.get(w.dtype)
    if dt is None or len(shape) != 1 or shape[0] != hd or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{hd}] of bfloat16, float16 or float32")
    return dt


def _table(table, kv_len, B, name="table", lengths="kv_len"):
    """Stride and width of a page table [B, pages]; checks the lengths too."""
    shape = table.shape
    if len(shape) != 2 or shape[0] != B:
        raise ValueError(f"{name} must be [{B}, pages]")
    st = table.stride()
    if table.dtype != torch.int32 or (shape[1] > 1 and st[1] != 1):
        raise ValueError(f"{name} must be int32 with a contiguous last axis")
    _vector(lengths, kv_len, B)
    if shape[1] > _INT_MAX:
        _size("pages of a table's row", shape[1])
    return st[0], shape[1]


def _cache(k, v, k_s, v_s, dtype, hd):
    """The packed C view of a cache, and its key heads."""
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("k_cache and v_cache must both be [pages, page, kv_heads, hd]")
    if shape[3] != hd:
        raise ValueError(f"the cache's head size {shape[3]} is not the queries' {hd}")
    if k.dtype != v.dtype:
        raise ValueError("k_cache and v_cache must share a dtype")
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the last axis of the cache must be contiguous")
    if shape[0] > _INT_MAX or shape[2] > _INT_MAX:
        _size("pages and heads of the cache", max(shape))
    if k.dtype == dtype:
        if k_s is not None or v_s is not None:
            raise ValueError("a 16-bit cache has no scales")
        return _PAGED_KV.pack(k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], 0, 0, 0, 0, 0, 0,
                              0, 0, _DT[dtype], shape[0], shape[1]), shape[2]
    if k.dtype != torch.int8:
        raise ValueError(f"the cache must be int8 or {dtype}")
    if k_s is None or v_s is None:
        raise ValueError("an int8 cache needs its scales k_s and v_s")
    for name, s in (("k_s", k_s), ("v_s", v_s)):
        if s.dtype != torch.float32 or s.shape != shape[:3]:
            raise ValueError(f"{name} must be float32 {list(shape[:3])}")
    return _PAGED_KV.pack(k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], k_s.data_ptr(),
                          *k_s.stride(), v_s.data_ptr(), *v_s.stride(), QLIN_I8, shape[0], shape[1]), shape[2]


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
    the cache, stores nothing; the others must differ: what a slot given twice holds is of
    no one token).  An int8 cache gets codes round_half_away(y / s) with `s = max(amax / 127,
    1e-8)` of each token's head in k_s / v_s.  Returns q_out."""
    T, hq, hd, dt, qt, qh = _queries(q)
    kshape = k.shape
    if len(kshape) != 3:
        raise ValueError("k must be [rows, kv_heads, hd]")
    dtype, hkv = q.dtype, kshape[1]
    kt, kh = _strides("k", k, T, hkv, hd, dtype)
    qot, qoh = _strides("q_out", q_out, T, hq, hd, dtype)
    pshape, pst = pos.shape, pos.stride()
    if len(pshape) == 1:
        pshape, pst = (1, pshape[0]), (0, pst[0])
    if len(pshape) != 2 or pshape[1] != T:
        raise ValueError(f"pos must be [{T}] or [axes, {T}]")
    pdt, fdt, fshape = pos.dtype, freqs.dtype, freqs.shape
    pos64 = pdt is torch.int64
    if not pos64 and pdt is not torch.int32:
        raise ValueError("pos must be int32 or int64")
    freqs64 = fdt is torch.float64
    if len(fshape) != 1 or not (freqs64 or fdt is torch.float32) or not freqs.is_contiguous():
        raise ValueError("freqs must be a contiguous float32 or float64 vector")
    half, axes = fshape[0], pshape[0]
    if sections is None:
        if axes != 1:
            raise ValueError(f"{axes} position axes need sections")
        sections = (half,)
    if len(sections) != axes:
        raise ValueError(f"sections must give one length for each of the {axes} axes")
    if axes > 3:
        raise ValueError("at most 3 position axes")
    wdt = qwp = kwp = 0
    if q_w is not None:
        wdt, qwp = _weight("q_w", q_w, hd), q_w.data_ptr()
    if k_w is not None:
        kdt, kwp = _weight("k_w", k_w, hd), k_w.data_ptr()
        if wdt and wdt != kdt:
            raise ValueError("q_w and k_w must share a dtype")
        wdt = kdt
    kop = kot = koh = vp = vt = vh = sp = slots64 = 0
    cache = None
    if k_out is not None:
        kot, koh = _strides("k_out", k_out, T, hkv, hd, dtype)
        kop = k_out.data_ptr()
    if k_cache is not None or v_cache is not None or slots is not None:
        if k_cache is None or v_cache is None or v is None or slots is None:
            raise ValueError("a cache takes k_cache, v_cache, v and slots")
        vt, vh = _strides("v", v, T, hkv, hd, dtype)
        _vector("slots", slots, T, _INTS)
        vp, sp, slots64 = v.data_ptr(), slots.data_ptr(), slots.dtype is torch.int64
        cache, ch = _cache(k_cache, v_cache, k_s, v_s, dtype, hd)
        if ch != hkv:
            raise ValueError(f"the cache has {ch} key heads, k {hkv}")
    elif k_out is None:
        raise ValueError("give k_out, a cache, or both")
    C.require_cuda(q, k, v, pos, freqs, q_out, k_out, k_cache, v_cache, slots, k_s, v_s, q_w, k_w)
    dev = q.get_device()
    s0, s1, s2 = (*sections, 0, 0)[:3]
    args = _ROPE.pack(
        q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, vp, vt, vh, q_out.data_ptr(), qot, qoh, kop, kot, koh, sp, slots64,
        pos.data_ptr(), pst[0], pst[1], pos64, freqs.data_ptr(), freqs64, qwp, kwp, wdt, bool(one_plus), eps, T, hq,
        hkv, hd, 2 * half, axes, s0, s1, s2, bool(interleaved), dt)
    _call("qlin_qk_norm_rope", dev, args, cache, C.current_stream(dev))
    return q_out


def attn_prompt(q, k, v, cu_q, out, cu_k=None, scale=None, causal=True):
    """Attention of packed prompts: sequence b's queries are rows cu_q[b] .. cu_q[b + 1] - 1
    of q [T, q_heads, hd], its keys and values rows cu_k[b] .. (default: cu_q) of k, v
    [Tk, kv_heads, hd].  cu_q, cu_k: int32 [B + 1], rising from 0.  `causal`: query i of a
    sequence sees its keys j <= i + keys - queries (the last query sees all).  scale (a
    positive number): hd ** -0.5 unless given.  out [T, q_heads, hd]; a row that sees no key is zero, rows of
    no sequence stay as they were.  Returns out."""
    T, hq, hd, dt, qt, qh = _queries(q)
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError("k and v must both be [rows, kv_heads, hd]")
    Tk, hkv = _size("rows of k", k.shape[0]), _size("heads of k", k.shape[1])
    kt, kh = _strides("k", k, Tk, hkv, hd, q.dtype)
    vt, vh = _strides("v", v, Tk, hkv, hd, q.dtype)
    ot, oh = _strides("out", out, T, hq, hd, q.dtype)
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must be [sequences + 1]")
    B = _size("sequences", cu_q.shape[0] - 1)
    _vector("cu_q", cu_q, B + 1)
    if cu_k is None:
        if Tk != T:
            raise ValueError("k and v must have the queries' rows, or cu_k be given")
        cu_k = cu_q
    else:
        _vector("cu_k", cu_k, B + 1)
    C.require_cuda(q, k, v, cu_q, cu_k, out)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_prompt", out.get_device(), q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
          cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), ot, oh, T, Tk, B, hq, hkv, hd, dt,
          hd ** -0.5 if scale is None else scale, bool(causal), ws, nws, stream)
    return out


def attn_prompt_paged(q, k_cache, v_cache, table, kv_len, cu_q, out, k_s=None, v_s=None, scale=None, causal=True):
    """`attn_prompt` over the cache, for a chunk of each prompt: sequence b's keys are the
    first kv_len[b] tokens of pages table[b, 0], table[b, 1], ... (its chunk's own among
    them: store them first).  table: int32 [B, pages a sequence], kv_len: int32 [B], cu_q:
    int32 [B + 1].  Returns out."""
    T, hq, hd, dt, qt, qh = _queries(q)
    cache, hkv = _cache(k_cache, v_cache, k_s, v_s, q.dtype, hd)
    ot, oh = _strides("out", out, T, hq, hd, q.dtype)
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must be [sequences + 1]")
    B = _size("sequences", cu_q.shape[0] - 1)
    _vector("cu_q", cu_q, B + 1)
    tb, pages = _table(table, kv_len, B)
    C.require_cuda(q, k_cache, v_cache, table, kv_len, cu_q, out, k_s, v_s)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_prompt_paged", out.get_device(), q.data_ptr(), qt, qh, cache, table.data_ptr(), tb, pages,
          kv_len.data_ptr(), cu_q.data_ptr(), out.data_ptr(), ot, oh, T, B, hq, hkv, hd, dt,
          hd ** -0.5 if scale is None else scale, bool(causal), ws, nws, stream)
    return out


def attn_decode(q, k_cache, v_cache, table, kv_len, out, k_s=None, v_s=None, scale=None):
    """Attention of one new token of each sequence: q and out [B, q_heads, hd]; sequence b's
    keys are the first kv_len[b] tokens (the new one among them) of pages table[b, 0],
    table[b, 1], ...  table: int32 [B, pages a sequence], kv_len: int32 [B].  A sequence
    without keys gives zeros.  scale: hd ** -0.5 unless given.  Returns out."""
    B, hq, hd, dt, qb, qh = _queries(q)
    cache, hkv = _cache(k_cache, v_cache, k_s, v_s, q.dtype, hd)
    ob, oh = _strides("out", out, B, hq, hd, q.dtype)
    tb, pages = _table(table, kv_len, B)
    C.require_cuda(q, k_cache, v_cache, table, kv_len, out, k_s, v_s)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_decode", out.get_device(), q.data_ptr(), qb, qh, cache, table.data_ptr(), tb, pages,
          kv_len.data_ptr(), out.data_ptr(), ob, oh, B, hq, hkv, hd, dt, hd ** -0.5 if scale is None else scale, ws,
          nws, stream)
    return out


def attn_decode_shared(q, k_cache, v_cache, prefix_table, prefix_len, cu_seq, table, kv_len, out, k_s=None, v_s=None,
                       scale=None):
    """`attn_decode` for sequences in groups that share a prefix (the candidates of one prompt,
    prompts behind one instruction): q and out [B, q_heads, hd].  Group g's sequences are rows
    cu_seq[g] .. cu_seq[g + 1] - 1; each sees the first prefix_len[g] tokens of pages
    prefix_table[g, 0], prefix_table[g, 1], ..., whose keys are read once for the group, and
    then its own first kv_len[b] tokens (the new one among them) of pages table[b, 0], ...
    A prefix may end anywhere in its last page.  prefix_table: int32 [groups, pages],
    prefix_len: int32 [groups], cu_seq: int32 [groups + 1], rising from 0; table and kv_len as
    attn_decode's.  A sequence without keys gives zeros; rows behind the last group stay as
    they were.  scale: hd ** -0.5 unless given.  Returns out."""
    B, hq, hd, dt, qb, qh = _queries(q)
    cache, hkv = _cache(k_cache, v_cache, k_s, v_s, q.dtype, hd)
    ob, oh = _strides("out", out, B, hq, hd, q.dtype)
    G = cu_seq.numel() - 1
    if cu_seq.dim() != 1 or G < 0:
        raise ValueError("cu_seq must be [groups + 1]")
    _size("groups", G)
    _vector("cu_seq", cu_seq, G + 1)
    pb, ppages = _table(prefix_table, prefix_len, G, "prefix_table", "prefix_len")
    tb, pages = _table(table, kv_len, B)
    C.require_cuda(q, k_cache, v_cache, prefix_table, prefix_len, cu_seq, table, kv_len, out, k_s, v_s)
    ws, nws, stream = C.scratch(out)
    _call("qlin_attn_decode_shared", out.get_device(), q.data_ptr(), qb, qh, cache, prefix_table.data_ptr(), pb, ppages,
          prefix_len.data_ptr(), cu_seq.data_ptr(), G, table.data_ptr(), tb, pages, kv_len.data_ptr(), out.data_ptr(),
          ob, oh, B, hq, hkv, hd, dt, hd ** -0.5 if scale is None else scale, ws, nws, stream)
    return out
