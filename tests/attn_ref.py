"""64-bit forms of the attention layer's middle, and how far a kernel may be from them.

u is half a step of a type relative to the value (`finfo.eps / 2`).  A kernel rounds

* its output once: u |o|;
* P (times a value's scale, where the cache is int8) to 16 bits for its product: u_p A, with
  A = sum_j p_j |v_j| / sum_j p_j, as each term moves by at most u_p of itself; u_p is that of the
  queries' type, of bf16 in prompts of bf16 queries over int8, and 2^-16 where P goes as two bf16
  numbers (decode and fp16 queries over int8);
* in 32 bits (e = 2^-24): a score's hd products and sums, (hd + 4) e S with
  S = scale max_j sum_d |q_d k_jd| (every p moves by a factor exp(+-that) and their sum too, hence
  twice), exponentials and rescaling (16 e), and sums over n keys of which no accumulator takes
  more than n / 8 steps: (n / 8 + 64) e, once for the sum of P and once for O.
"""
from __future__ import annotations

import torch

E32 = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def attend(q, k, v, scale, seen, dt, up=None):
    """q [Lq, HQ, D], k / v [Lk, HKV, D] of any type, seen [Lq, Lk] (bool).  Returns the
    output and the allowed error, both in 64 bits, [Lq, HQ, D]."""
    lq, hq, d = q.shape
    lk, hkv = k.shape[:2]
    out = torch.zeros((lq, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u = half_step(dt)
    up = u if up is None else up
    if lk == 0 or lq == 0:
        return out, tol + 1e-30
    some = seen.any(1)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)].double(), v[:, h // (hq // hkv)].double()
        qh = q[:, h].double()
        s = (qh @ kh.t() * scale).masked_fill(~seen, -torch.inf)
        m = torch.where(some, s.amax(1), 0.0)
        p = torch.exp(s - m[:, None])
        p = torch.where(seen, p, 0.0)
        l = torch.where(some, p.sum(1), 1.0)[:, None]
        # (a masked value has no part whatever it holds)
        o = (p @ torch.nan_to_num(vh, nan=0.0, posinf=0.0, neginf=0.0)) / l
        a = (p @ torch.nan_to_num(vh, nan=0.0, posinf=0.0, neginf=0.0).abs()) / l
        S = (qh.abs() @ kh.abs().t() * scale).masked_fill(~seen, 0.0).nan_to_num(0.0, 0.0, 0.0).amax(1, keepdim=True)
        t = u * o.abs() + a * (up + 2 * (d + 4) * E32 * S + (16 + 2 * (lk / 8 + 64)) * E32)
        out[:, h], tol[:, h] = torch.where(some[:, None], o, 0.0), t * 1.01 + 1e-30
    # a subnormal fp16 output is off by half its spacing instead
    if dt == torch.float16:
        tol += 2.0 ** -25
    return out, tol


def causal(lq, lk, device):
    i = torch.arange(lq, device=device)[:, None]
    return torch.arange(lk, device=device)[None, :] <= i + lk - lq


def check(y, ref, tol, name=""):
    y = y.double()
    err = (y - ref).abs()
    bad = ~(err <= tol)
    if bad.any():
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of tolerance, first at {at}: "
                             f"{float(y[at])} against {float(ref[at])} +- {float(tol[at]):.3e}")


def pages_of(lens, page, spare, seed, device="cpu"):
    """A shuffled page table [B, most pages (+ 1)], and the number of pages; entries behind a
    sequence's end name no page."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table.to(device), pages


def cache(pages, page, hkv, hd, dt, seed, int8=False, head_major=True, device="cuda"):
    """A cache of random values (k, v, k_s, v_s), [pages, page, hkv, hd]."""
    g = torch.Generator(device=device).manual_seed(seed)
    shape = (pages, hkv, page, hd) if head_major else (pages, page, hkv, hd)
    turn = (lambda x: x.transpose(1, 2)) if head_major else (lambda x: x)
    if not int8:
        return (*(turn(torch.randn(shape, generator=g, device=device).to(dt)) for _ in range(2)), None, None)
    k, v = (turn(torch.randint(-127, 128, shape, generator=g, device=device, dtype=torch.int8)) for _ in range(2))
    ks, vs = (turn(torch.rand(shape[:3], generator=g, device=device) * 0.02 + 0.002) for _ in range(2))
    return k, v, ks, vs


def gathered(c, table, b, n):
    """The first n keys and values of sequence b, as 64-bit numbers, [n, hkv, hd]."""
    k, v, ks, vs = c
    page = k.shape[1]
    ids = table[b, :-(-n // page)].long()
    out = []
    for x, s in ((k, ks), (v, vs)):
        y = x[ids].reshape(-1, *x.shape[2:])[:n].double()
        if s is not None:
            y = y * s[ids].reshape(-1, x.shape[2])[:n, :, None].double()
        out.append(y)
    return out
