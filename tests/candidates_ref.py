"""64-bit forms of a decode step of several candidates beside its linears, and how far a kernel
may be from them (attn_ref.py for attention's)."""
from __future__ import annotations

import math

import attn_ref as R
import torch

E32 = 2.0 ** -24


# ------------------------------------------------------------------ attention over shared prefixes

class Batch:
    """Groups of sequences over one cache: `groups` [(sequences, prefix keys)], `own` keys of each
    sequence, `pad` rows behind the last group."""

    def __init__(self, groups, own, hq, hkv, hd, dt, seed, page=64, int8=False, pad=0, head_major=True, device="cuda",
                 scale=None):
        self.groups, self.own, self.hkv, self.dt = groups, own, hkv, dt
        self.scale = hd ** -0.5 if scale is None else scale
        B = sum(n for n, _ in groups)
        assert len(own) == B
        lens = [p for _, p in groups] + own + [0] * pad
        table, pages = R.pages_of(lens, page, 3, seed, device)
        G = len(groups)
        self.ptable, self.table = table[:G].contiguous(), table[G:].contiguous()
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        self.plen, self.len = ints([p for _, p in groups]), ints(own + [0] * pad)
        self.cu = ints([sum(n for n, _ in groups[:i]) for i in range(G + 1)])
        self.cache = R.cache(pages, page, hkv, hd, dt, seed + 1, int8, head_major, device)
        g = torch.Generator(device=device).manual_seed(seed + 2)
        self.q = (torch.randn((B + pad, hq, hd), generator=g, device=device) * 2).to(dt)
        self.out = torch.full_like(self.q, 7.0)

    def run(self, out=None, **kw):
        from qwen35_amd.kernels import attention as A
        k, v, ks, vs = self.cache
        args = dict(q=self.q, prefix_table=self.ptable, prefix_len=self.plen, cu_seq=self.cu, table=self.table,
                    kv_len=self.len, out=self.out if out is None else out) | kw
        return A.attn_decode_shared(args.pop("q"), k, v, **args, k_s=ks, v_s=vs, scale=self.scale)

    def expected(self):
        """Outputs and allowed errors of the groups' rows."""
        outs, tols, b = [], [], 0
        up = 2.0 ** -16 if self.cache[2] is not None else None
        for g, (n, p) in enumerate(self.groups):
            kp, vp = R.gathered(self.cache, self.ptable, g, p)
            for _ in range(n):
                ko, vo = R.gathered(self.cache, self.table, b, self.own[b])
                k, v = torch.cat([kp, ko]), torch.cat([vp, vo])
                seen = torch.ones((1, len(k)), dtype=torch.bool, device=k.device)
                o, t = R.attend(self.q[b:b + 1], k, v, self.scale, seen, self.dt, up)
                outs.append(o)
                tols.append(t)
                b += 1
        if not outs:
            z = torch.zeros((0, *self.q.shape[1:]), dtype=torch.float64, device=self.q.device)
            return z, z
        return torch.cat(outs), torch.cat(tols)

    def check(self, y, name=""):
        ref, tol = self.expected()
        R.check(y[:len(ref)], ref, tol, name)


# ------------------------------------------------------------------ logits

def logits_formula(x, tokens=None, lens=None, prompt=None, rep=1.0, pres=0.0, freq=0.0, ids=None, bias=None, allowed=None,
                   to=torch.float64):
    """Row by row in lists and 64 bits; the allowed error counts half a step of 32 bits of every number on
    the way (relative to its size), and of the output's type."""
    B, V = x.shape
    row = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else v
    out, tol = x.double().cpu().clone(), torch.zeros((B, V), dtype=torch.float64)
    for b in range(B):
        y, t = out[b], tol[b]
        if tokens is not None:
            h = tokens[b].tolist()
            n = len(h) if lens is None else min(max(int(lens[b]), 0), len(h))
            p = 0 if prompt is None else int(prompt[b])
            count, seen = {}, set()
            for i, tok in enumerate(h[:n]):
                if 0 <= tok < V:
                    seen.add(tok)
                    if i >= p:
                        count[tok] = count.get(tok, 0) + 1
            for tok in seen:
                v = float(y[tok])
                v = v / row(rep, b) if v > 0 else v * row(rep, b)
                e = abs(v)
                c = count.get(tok, 0)
                if c:
                    f = row(freq, b) * c
                    e += abs(f) + abs(v - f)
                    v -= f
                    v -= row(pres, b)
                    e += abs(v)
                y[tok], t[tok] = v, e * E32
        if ids is not None:
            last = {int(i): float(w) for i, w in zip(ids[b].tolist(), bias[b].tolist())}
            for tok, w in last.items():
                if 0 <= tok < V:
                    y[tok] += w
                    t[tok] += abs(float(y[tok])) * E32
        if allowed is not None:
            y[~allowed[b].cpu()] = -math.inf
    if to != torch.float32:
        # (half a step of a subnormal fp16 number is 2^-25)
        tol += torch.where(out.isfinite(), out.abs(), 0.0) * R.half_step(to) * 1.01 + (2.0 ** -25 if to == torch.float16 else 0.0)
    return out, tol * 1.01


def bits_of(allowed):
    """bool [B, V] as int32 words, the lowest bit first."""
    B, V = allowed.shape
    W = (V + 31) // 32
    a = torch.zeros((B, W * 32), dtype=torch.int64)
    a[:, :V] = allowed.long().cpu()
    w = (a.view(B, W, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32).to(allowed.device)


# ------------------------------------------------------------------ drawing

def draw(x, u, k, t=1.0, top_p=1.0, min_p=0.0):
    """(token, log probability, distance of the draw from the nearest border) of one row in 64 bits."""
    x = [float(v) for v in x.double().tolist()]
    order = sorted((i for i in range(len(x)) if x[i] > -math.inf), key=lambda i: (-x[i], i))
    if not order:
        return -1, -math.inf, 1.0
    top = order[:k]
    m = x[order[0]]

    def weight(v, t):
        if v == m:
            return 1.0
        if m == math.inf or t == 0:
            return 0.0
        return math.exp((v - m) / t)

    w = [weight(x[i], t) for i in top]
    total, kept, before, near = math.fsum(w), [], 0.0, 1.0
    for i, z in enumerate(w):
        near = min(near, abs(before - top_p * total) / total if i and top_p < 1 else 1.0)
        if i and not (before < top_p * total and z >= min_p):
            break
        kept.append(z)
        before += z
    goal, run = u * math.fsum(kept), 0.0
    at = len(kept) - 1
    for i, z in enumerate(kept):
        run += z
        near = min(near, abs(run - goal) / total)
        if run > goal:
            at = i
            break
    tok = top[at]
    full = math.fsum(weight(x[i], 1.0) for i in order)
    return tok, (0.0 if x[tok] == m else x[tok] - m) - math.log(full), near
