"""From the vocabulary head's rows to the next tokens.

The reference's sampler.py does this per row on the host's clock, with torch calls and a
synchronization for each token (sample_logits 20-80, sample_batch 83-125), under masks of
its section grammar (targets.py 102-198).  Here it is two launches that wait for nothing:

* `logits_process`  penalties for repeated tokens, biases and a mask of allowed tokens;
* `sample`          one token of each row, and its log probability.

A step of several candidates, from the vocabulary head to the next tokens:

    gemm_i8(aq, a_s, head, head_s, logits)                       # bf16 [B, V]
    logits_process(logits, scores, tokens=history, lens=lens, prompt_lens=prompt_lens,
                   repetition=1.1, mask=allowed)                 # float32 [B, V]
    sample(scores, u, tokens, logprobs=logprobs, temperature=0.7, top_k=20, top_p=0.8)

Numbers that a batch's requests have each their own of (penalties, temperature, top_p, min_p)
are floats or float32 tensors [B].  Histories, lengths, masks and these tensors stay on the
device and are never waited for; what they may hold is stated in include/qlin_candidates.h.  What a
call writes shares no memory with what it reads (`logits_process` in place aside).  All calls
run on the current stream of their tensors' device and can be captured (see `qlin.capture`).
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import qlin as C
from .attention import _INT_MAX, _call, _size, _vector
from .attention import _SIGS as _ALL

__all__ = ["logits_process", "sample"]

_P, _I, _L, _S, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float

_SIGS = {
    "qlin_logits_process": [ctypes.c_char_p, _P],
    "qlin_sample": [_P, _I, _L, _I, _I, _I, _P, _P, _F, _P, _F, _P, _F, _P, _I, _P, _P, _S, _P],
}
_ALL.update(_SIGS)
EXPORTS = ("qlin_attn_decode_shared", *_SIGS)  # of include/qlin_candidates.h

# include/qlin_candidates.h qlin_logits: logits, out and tokens with a stride; lengths; penalties; biases;
# the mask; sizes and types; penalties of all rows
_LOGITS = struct.Struct("@" + 3 * "Pq" + "2P3P" + 3 * "Pq" + "8i3f0q")

_FLOATS = {torch.bfloat16: C.QLIN_BF16, torch.float16: C.QLIN_F16, torch.float32: C.QLIN_F32}
_INTS = (torch.int32, torch.int64)


def _rows(name, t, B=None, n=None, dtypes=None):
    """Row stride of a matrix whose rows are contiguous."""
    shape = t.shape
    if len(shape) != 2 or (B is not None and shape[0] != B) or (n is not None and shape[1] != n):
        want = ", ".join("rows" if x is None else str(x) for x in (B, n))
        raise ValueError(f"{name} must be [{want}], not {list(shape)}")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}")
    st = t.stride()
    if shape[1] > 1 and st[1] != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")
    return st[0]


def _logit_rows(name, t):
    """Type code, row stride, rows and tokens."""
    dt, shape = _FLOATS.get(t.dtype), t.shape
    if dt is None:
        raise ValueError(f"{name} must be bfloat16, float16 or float32")
    if len(shape) != 2:
        raise ValueError(f"{name} must be [rows, tokens], not {list(shape)}")
    st = t.stride()
    if shape[1] > 1 and st[1] != 1:
        raise ValueError(f"the last axis of {name} must be contiguous")
    if shape[0] > _INT_MAX or shape[1] > _INT_MAX:
        _size(f"rows and tokens of {name}", max(shape))
    return dt, st[0], shape[0], shape[1]


def _value(name, x, B):
    """(address, number) of a float or a float32 tensor [B]."""
    if type(x) is float:
        return 0, x
    if isinstance(x, torch.Tensor):
        _vector(name, x, B, (torch.float32,))
        return x.data_ptr(), 1.0  # (a vector of no rows has no address: the number, one that all arguments may be, is checked)
    return 0, float(x)


def _tensor(x):
    return None if type(x) is float or not isinstance(x, torch.Tensor) else x


def logits_process(logits, out, tokens=None, lens=None, prompt_lens=None, repetition=1.0, presence=0.0, frequency=0.0,
                   bias_ids=None, bias=None, mask=None):
    """Penalties, biases and a mask on rows of logits [B, V] (bfloat16, float16 or float32), in
    32 bits, into out [B, V] (any of these types; may be logits itself).

    tokens: int32 or int64 [B, history], the tokens of each row so far; of them the first lens[b]
    count (int32 [B]; default: all), and of those the first prompt_lens[b] (default: none) are the
    prompt's.  A token among them is divided by `repetition` where its logit is positive and
    multiplied where not; one that comes c > 0 times behind the prompt loses `frequency` * c and
    then `presence`.  bias_ids int32 and bias float32 [B, n]: what is added to some tokens (of an
    id given twice the last counts).  mask: the allowed tokens, bits of int32 words
    [B, (V + 31) // 32] (token i is bit i % 32 of word i // 32) or bool [B, V]; others become -inf.
    An expanded row (stride 0) is one for all.  Ids outside the vocabulary, as padding
    has, count for nothing.  Returns out."""
    xdt, xs, B, V = _logit_rows("logits", logits)
    odt = _FLOATS.get(out.dtype)
    if odt is None:
        raise ValueError("out must be bfloat16, float16 or float32")
    os = _rows("out", out, B, V)
    rep, pres, freq = (_value(n, x, B) for n, x in (("repetition", repetition), ("presence", presence),
                                                    ("frequency", frequency)))
    tp = ts = t64 = L = lp = pp = 0
    if tokens is not None:
        ts = _rows("tokens", tokens, B, None, _INTS)
        tp, t64, L = tokens.data_ptr(), tokens.dtype is torch.int64, _size("tokens of a history", tokens.shape[1])
        if lens is not None:
            _vector("lens", lens, B)
            lp = lens.data_ptr()
        if prompt_lens is not None:
            _vector("prompt_lens", prompt_lens, B)
            pp = prompt_lens.data_ptr()
    elif lens is not None or prompt_lens is not None or rep != (0, 1.0) or pres != (0, 0.0) or freq != (0, 0.0):
        raise ValueError("penalties and lengths need tokens")
    ip = ist = bp = bst = nb = mp = mst = by_bytes = 0
    if bias is not None or bias_ids is not None:
        if bias is None or bias_ids is None:
            raise ValueError("biases take bias_ids and bias")
        ist = _rows("bias_ids", bias_ids, B, None, (torch.int32,))
        nb = _size("biases of a row", bias_ids.shape[1])
        bst = _rows("bias", bias, B, nb, (torch.float32,))
        ip, bp = bias_ids.data_ptr(), bias.data_ptr()
    if mask is not None:
        by_bytes = mask.dtype is torch.bool
        mst = _rows("mask", mask, B, V if by_bytes else (V + 31) // 32, (torch.bool, torch.int32))
        mp = mask.data_ptr()
    C.require_cuda(logits, out, tokens, lens, prompt_lens, _tensor(repetition), _tensor(presence), _tensor(frequency),
                   bias_ids, bias, mask)
    dev = out.get_device()
    args = _LOGITS.pack(logits.data_ptr(), xs, out.data_ptr(), os, tp, ts, lp, pp, rep[0], pres[0], freq[0], ip, ist, bp,
                        bst, mp, mst, t64, by_bytes, B, V, L, nb, xdt, odt, rep[1], pres[1], freq[1])
    _call("qlin_logits_process", dev, args, C.current_stream(dev))
    return out


def sample(logits, u, tokens, logprobs=None, temperature=1.0, top_k=20, top_p=1.0, min_p=0.0):
    """One token of each row of logits [B, V] (bfloat16, float16 or float32), into tokens (int64 or
    int32 [B]), by the uniform numbers u (float32 [B], 0 <= u < 1).

    Of the row's top_k largest logits (1 to 128; equal ones by their index) with the weights
    exp((x - max) / temperature), those are kept that have less than top_p of the weights' sum in
    front of them and weigh at least min_p of the largest; the first is drawn with which the sum of
    the kept exceeds u times theirs.  temperature 0 takes the largest, of equal ones the lowest index,
    whatever u is (only infinite logits share the row there too).  logprobs (float32 [B]): the
    token's log probability among all of the row's logits, as they are (at temperature 1).  Logits of
    -inf and NaN are never drawn; a row of nothing else gives -1 (and -inf).  Returns tokens."""
    xdt, xs, B, V = _logit_rows("logits", logits)
    _vector("u", u, B, (torch.float32,))
    _vector("tokens", tokens, B, _INTS)
    lp = 0
    if logprobs is not None:
        _vector("logprobs", logprobs, B, (torch.float32,))
        lp = logprobs.data_ptr()
    (tp, t), (pp, p), (mp, m) = (_value(n, x, B) for n, x in (("temperature", temperature), ("top_p", top_p),
                                                              ("min_p", min_p)))
    C.require_cuda(logits, u, tokens, logprobs, _tensor(temperature), _tensor(top_p), _tensor(min_p))
    ws, nws, stream = C.scratch(tokens)
    _call("qlin_sample", tokens.get_device(), logits.data_ptr(), xdt, xs, B, V, _size("top_k", top_k), u.data_ptr(), tp, t,
          pp, p, mp, m, tokens.data_ptr(), tokens.dtype is torch.int64, lp, ws, nws, stream)
    return tokens
