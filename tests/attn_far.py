"""One row of attention over very many keys in 64 bits, and how far a kernel may be from it.

u = half a step of the type, e = 2^-24, A = sum_j p_j |v_j| / sum_j p_j, S = scale max_j |q| . |k_j|:

* the output's rounding u |o| (2^-25 where an fp16 one is subnormal) and P's u_p A;
* 32 bits: a score's products and sums move every p by a factor exp(+-(hd + 4) e S), exponentials and
  rescaling by 16 e, sums by `adds` e for O and for the sum of P each.  `adds` bounds the additions that one
  value goes through: 32 keys of a product, a unit's blocks a wave, the joins of waves and parts;
* fp16: keys of the heaviest one's block are taken against a reference that puts it at 2^8 at least, where
  a subnormal is off by at most 2^-25: 32 2^-33 of its P, of the largest value.
"""
from __future__ import annotations

import torch

import attn_ref as R

# calls over the cache: 8 of 32 blocks a wave in decode steps, at most 2^15 / 192 = 171 in prompts at 2^20
# keys, at most 448 + 4 joins
ADDS = 32 + 171 + 452


def row(q, k, v, dt, up=None, adds=ADDS):
    """q [G, hd], k / v [n, hd] (one key head).  Returns the output, the allowed error [G, hd] and the
    keys' weights [G, n]."""
    hd = q.shape[-1]
    scale, u = hd ** -0.5, R.half_step(dt)
    qd, kd, vd = q.double(), k.double(), v.double()
    s = qd @ kd.t() * scale
    p = torch.exp(s - s.amax(1, keepdim=True))
    l = p.sum(1, keepdim=True)
    o, A = p @ vd / l, p @ vd.abs() / l
    S = (qd.abs() @ kd.abs().t() * scale).amax(1, keepdim=True)
    tol = u * o.abs() + A * ((u if up is None else up) + 2 * (hd + 4) * R.E32 * S + (16 + 2 * adds) * R.E32)
    if dt == torch.float16:
        tol = tol + 2.0 ** -25 + 32 * 2.0 ** -33 / l * vd.abs().max()
    return o, tol, p / l


def paged(k, v, page, seed, int8=False):
    """k, v [n, hd] in pages of a cache of one key head, in any order: the cache (k, v, k_s, v_s) and the table."""
    n, pages = k.shape[0], -(-k.shape[0] // page)
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None]
    i = torch.arange(n, device="cuda")
    at, off = table[0].long()[i // page], i % page
    out, scales = [], []
    for x in (k, v):
        c = torch.zeros((pages, page, 1, x.shape[1]), dtype=torch.int8 if int8 else x.dtype, device="cuda")
        s = torch.zeros((pages, page, 1), device="cuda")
        if int8:
            s[at, off, 0] = x.float().abs().amax(1) / 127
            x = (x.float() / s[at, off]).round().to(torch.int8)
        c[at, off, 0] = x
        out.append(c)
        scales.append(s if int8 else None)
    return (*out, *scales), table
