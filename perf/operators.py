"""Operators between an attention layer's projections, and how their speed is watched.

The engine's attention layer projects (proj3), normalises and rotates queries and keys
and stores keys and values in the cache, attends, and multiplies by the gates
(gate_mul_quant) into the output projection.  The cases are the work in the middle:

* rope     per-head RMSNorm of queries and keys, rotary positions of one or three axes
           on the leading part of a head, keys and values into a paged cache
           (16-bit, or int8 with a scale for each token and head);
* prompt   attention of packed prompts over their own keys, causal;
* chunk    attention of the next chunk of a prompt over the paged cache, causal;
* decode   attention of one new token of each sequence over the paged cache.

A case is a dict of plain values.  `prepare(case, seed)` makes inputs and buffers on the
GPU, `run(state)` is one pass, `exact(case, seed)` the same in 64 bits, `work(case)` the
bytes and operations a pass cannot do without.  `own` picks the plain torch form or the
package's kernels.
"""
from __future__ import annotations

import importlib
import importlib.util
import math
import pathlib
import random
import sys

import torch

own = False

ALIAS = "qwen35_amd"
ROOT = pathlib.Path(__file__).resolve().parent.parent
EPS = 1e-6
THETA = 1e7
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _attention():
    """The package's kernels.attention; its directory is no Python identifier, so it is
    loaded under an alias."""
    if ALIAS not in sys.modules:
        pkg = ROOT / "qwen_3.5_comfy_prompt_enhancer_amd"
        spec = importlib.util.spec_from_file_location(ALIAS, pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[ALIAS] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module(f"{ALIAS}.kernels.attention")


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # the smallest call: one token of one sequence, on its way into a decode step
        dict(name="rope-1", kind="rope", T=1, HQ=8, HKV=2, HD=256, rot=64, axes=1, inter=False, dt="bf16",
             kv="16", page=64),
        # a prompt chunk with an image in it: time, height and width positions
        dict(name="rope-512-3axes", kind="rope", T=512, HQ=8, HKV=2, HD=256, rot=64, axes=3, inter=True,
             dt="bf16", kv="16", page=64),
        # several packed prompts of a larger model into an int8 cache, an odd number of tokens
        dict(name="rope-4097-int8", kind="rope", T=4097, HQ=16, HKV=4, HD=256, rot=64, axes=3, inter=False,
             dt="bf16", kv="int8", page=16),
        # one prefill chunk, the first of its prompt
        dict(name="prompt-512", kind="prompt", B=1, L=512, even=True, mix=0, HQ=8, HKV=2, HD=256, dt="bf16"),
        # a batch of prompts of different lengths, one of them empty, fp16, smaller heads
        dict(name="prompt-packed-9x1500", kind="prompt", B=9, L=1500, even=False, mix=3, HQ=16, HKV=2, HD=128,
             dt="fp16"),
        # the longest prompt the engine takes, in one piece
        dict(name="prompt-8192", kind="prompt", B=1, L=8192, even=True, mix=0, HQ=8, HKV=2, HD=256, dt="bf16"),
        # a later chunk of a long prompt, over an int8 cache
        dict(name="chunk-512-past-6000-int8", kind="chunk", B=1, L=512, past=6000, mix=1, HQ=8, HKV=2, HD=256,
             dt="bf16", kv="int8", page=64),
        # four prompts' chunks of different lengths and pasts, small pages
        dict(name="chunk-4x700-past-3000", kind="chunk", B=4, L=700, past=3000, mix=2, HQ=16, HKV=4, HD=256,
             dt="bf16", kv="16", page=16),
        # token generation of one sequence early in its answer
        dict(name="decode-1x1000", kind="decode", B=1, L=1000, even=True, mix=0, HQ=8, HKV=2, HD=256, dt="bf16",
             kv="16", page=64),
        # eight candidates of a long prompt, of different lengths
        dict(name="decode-8x8192", kind="decode", B=8, L=8192, even=False, mix=4, HQ=16, HKV=4, HD=256,
             dt="bf16", kv="16", page=64),
        # one sequence with a very long context in int8
        dict(name="decode-1x131072-int8", kind="decode", B=1, L=131071, even=True, mix=0, HQ=8, HKV=2, HD=256,
             dt="bf16", kv="int8", page=64),
        # a full serving batch, fp16, smaller heads, eight query heads to a key head
        dict(name="decode-64x16384", kind="decode", B=64, L=16384, even=False, mix=5, HQ=32, HKV=4, HD=128,
             dt="fp16", kv="16", page=32),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["rope", "prompt", "prompt", "chunk", "decode", "decode"])
    hkv = rng.choice([1, 2, 4, 5])
    hd = rng.choice([64, 128, 256, 256])
    c = dict(kind=kind, HQ=hkv * rng.choice([1, 3, 4, 4, 8]), HKV=hkv, HD=hd, dt=rng.choice(["bf16", "bf16", "fp16"]))
    mix = rng.randrange(1, 1 << 20)
    if kind != "prompt":
        c |= dict(kv=rng.choice(["16", "16", "int8"]), page=rng.choice([16, 32, 64, 128]))
    if kind == "rope":
        axes = rng.choice([1, 3])
        return c | dict(T=_log(rng, 1, 8192), rot=rng.choice([32, 64, hd]) if hd > 64 else 64, axes=axes,
                        inter=axes == 3 and rng.random() < 0.5)
    # scores of a pass: query heads x queries x keys, at most what the longest listed prompt has
    if kind == "prompt":
        b = _log(rng, 1, 16)
        return c | dict(B=b, L=min(_log(rng, 1, 8192), int(8192 * math.sqrt(8 / c["HQ"] / b))),
                        even=rng.random() < 0.3, mix=mix)
    if kind == "chunk":
        b, n = _log(rng, 1, 8), _log(rng, 1, 700)
        return c | dict(B=b, L=n, past=min(_log(rng, 1, 16384), (1 << 27) // (c["HQ"] * b * n)), mix=mix)
    b = _log(rng, 1, 64)
    return c | dict(B=b, L=min(_log(rng, 1, 131072), 240_000_000 // (b * hkv * hd)), even=rng.random() < 0.3,
                    mix=mix)


def _lens(case):
    """(queries, keys) of each sequence.  Uneven batches: the first is the longest, one may be
    empty (a padded entry), the others lie in between."""
    b, top = case["B"], case["L"]
    rng = random.Random(case["mix"])
    if case["kind"] == "chunk":
        nq = [top if i == 0 else rng.randint(1, top) for i in range(b)]
        return nq, [n + (case["past"] if i == 0 else rng.randint(0, case["past"])) for i, n in enumerate(nq)]
    n = [top if i == 0 or case["even"] else rng.randint(1, top) for i in range(b)]
    if b > 2 and not case["even"]:
        n[1] = 0
    return ([1] * b if case["kind"] == "decode" else n), n


def work(case):
    hq, hkv, hd = case["HQ"], case["HKV"], case["HD"]
    kvb = hd * 2 if case.get("kv", "16") == "16" else hd + 4          # bytes of a token's key of one head
    if case["kind"] == "rope":
        t, r = case["T"], case["rot"]
        read = t * (hq + 2 * hkv) * hd * 2 + 2 * hd * 2 + t * 8 * (case["axes"] + 1) + r // 2 * 8
        return {"bytes": read + t * hq * hd * 2 + 2 * t * hkv * kvb, "flops": t * (hq + hkv) * (5 * hd + 3 * r)}
    nq, nk = _lens(case)
    if case["kind"] == "decode":
        pairs = sum(nk)
    else:
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(nq, nk))
    b = 2 * sum(nq) * hq * hd * 2 + 2 * sum(nk) * hkv * kvb + 4 * (len(nq) + 1)
    if case["kind"] != "prompt":
        b += 4 * sum(-(-n // case["page"]) for n in nk) + 4 * len(nk)
    return {"bytes": b, "flops": 4 * pairs * hq * hd}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1 + seed)


def _randn(g, shape, dt):
    return torch.randn(shape, generator=g, device="cuda").to(dt)


def _cache(g, case, pages):
    """Keys and values [pages, page, HKV, HD] (a page holds one head's tokens next to each other)."""
    shape = (pages, case["HKV"], case["page"], case["HD"])
    if case["kv"] == "16":
        k, v = (_randn(g, shape, DTYPES[case["dt"]]).permute(0, 2, 1, 3) for _ in range(2))
        return dict(k_cache=k, v_cache=v, k_s=None, v_s=None)
    k, v = (torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8).permute(0, 2, 1, 3)
            for _ in range(2))
    ks, vs = ((torch.rand(shape[:3], generator=g, device="cuda") * 0.02 + 0.005).permute(0, 2, 1) for _ in range(2))
    return dict(k_cache=k, v_cache=v, k_s=ks, v_s=vs)


def _cu(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dt"]]
    hq, hkv, hd = case["HQ"], case["HKV"], case["HD"]
    if case["kind"] == "rope":
        t, page, half = case["T"], case["page"], case["rot"] // 2
        # the projection's rows: each head's queries and gates, then keys, then values
        proj = _randn(g, (t, 2 * hq * hd + 2 * hkv * hd), dt)
        pages = t // page + 2
        # an image of a third of the tokens between text: its rows share a time, and its text goes on
        start = torch.randint(0, 200000, (1,), generator=g, device="cuda")
        i = torch.arange(t, device="cuda")
        a, b = t // 3, 2 * t // 3
        pic = (i >= a) & (i < b)
        w = max(1, int(math.isqrt(max(1, b - a))))
        pos = torch.stack([torch.where(pic, torch.full_like(i, a), i), torch.where(pic, a + (i - a) // w, i),
                           torch.where(pic, a + (i - a) % w, i)])[:case["axes"]] + start
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
        sections = [half] if case["axes"] == 1 else [half - 2 * (half // 3), half // 3, half // 3]
        st = dict(q=proj[:, :2 * hq * hd].view(t, hq, 2 * hd)[:, :, :hd],
                  k=proj[:, 2 * hq * hd:(2 * hq + hkv) * hd].view(t, hkv, hd),
                  v=proj[:, (2 * hq + hkv) * hd:].view(t, hkv, hd), pos=pos, slots=slots, sections=sections,
                  freqs=torch.tensor([THETA ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda"),
                  q_w=_randn(g, (hd,), dt) * 0.2, k_w=_randn(g, (hd,), dt) * 0.2,
                  q_out=torch.empty((t, hq, hd), dtype=dt, device="cuda"), **_cache(g, case, pages))
        return st | dict(case=case)
    nq, nk = _lens(case)
    st = dict(case=case, scale=hd ** -0.5, q=_randn(g, (sum(nq), hq, hd), dt) * 2,
              out=torch.empty((sum(nq), hq, hd), dtype=dt, device="cuda"), nq=max(nq), nk=max(nk))
    if case["kind"] != "decode":
        st["cu_q"] = _cu(nq)
    if case["kind"] == "prompt":
        # keys and values as columns of the projection's rows
        kv = _randn(g, (sum(nk), 2 * hkv * hd), dt)
        return st | dict(k=kv[:, :hkv * hd].view(-1, hkv, hd), v=kv[:, hkv * hd:].view(-1, hkv, hd))
    need = [-(-n // case["page"]) for n in nk]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda")[:sum(need)].to(torch.int32)
    table = torch.zeros((len(nk), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return st | dict(table=table, kv_len=torch.tensor(nk, dtype=torch.int32, device="cuda"),
                     **_cache(g, case, pages))


# ------------------------------------------------------------------ one pass

def _cache_values(st):
    """The caches as the values they stand for."""
    if st["k_s"] is None:
        return st["k_cache"], st["v_cache"]
    dt = st["q"].dtype
    return (st["k_cache"] * st["k_s"][..., None]).to(dt), (st["v_cache"] * st["v_s"][..., None]).to(dt)


def _own(st):
    A, c = _attention(), st["case"]
    cache = [st.get(n) for n in ("k_cache", "v_cache")]
    if c["kind"] == "rope":
        A.qk_norm_rope(st["q"], st["k"], st["pos"], st["freqs"], st["q_out"], v=st["v"], k_cache=cache[0],
                       v_cache=cache[1], slots=st["slots"], k_s=st["k_s"], v_s=st["v_s"], q_w=st["q_w"],
                       k_w=st["k_w"], eps=EPS, sections=st["sections"], interleaved=c["inter"])
        return [st["q_out"], *_cache_values(st)]
    if c["kind"] == "prompt":
        A.attn_prompt(st["q"], st["k"], st["v"], st["cu_q"], st["out"], scale=st["scale"])
    elif c["kind"] == "chunk":
        A.attn_prompt_paged(st["q"], *cache, st["table"], st["kv_len"], st["cu_q"], st["out"], k_s=st["k_s"],
                            v_s=st["v_s"], scale=st["scale"])
    else:
        A.attn_decode(st["q"], *cache, st["table"], st["kv_len"], st["out"], k_s=st["k_s"], v_s=st["v_s"],
                      scale=st["scale"])
    return [st["out"]]


def _axis_of(half, sections, interleaved, device):
    """The position axis of each frequency: runs of the sections' lengths, or axes in turn (an axis
    whose section is used up leaves its turns to the first)."""
    i = torch.arange(half, device=device)
    if not interleaved:
        ends = torch.tensor(sections, device=device).cumsum(0)
        return (i[:, None] >= ends[None, :-1]).sum(1)
    n = len(sections)
    room = torch.tensor(sections, device=device) * n
    return torch.where(i < room[i % n], i % n, 0)


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.float())


def _rotated(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _codes(x):
    """int8 codes (ties away from zero) and the scale of each token and head."""
    s = (x.abs().amax(-1) / 127).clamp_min(1e-8)
    r = x / s[..., None]
    return torch.trunc(r + torch.where(r >= 0, 0.5, -0.5)).clamp(-127, 127).to(torch.int8), s


def _plain_rope(st):
    c = st["case"]
    axis = _axis_of(c["rot"] // 2, st["sections"], c["inter"], "cuda")
    angle = st["pos"].to(torch.float64)[axis].t() * st["freqs"]              # [T, rot/2]
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    st["q_out"].copy_(_rotated(_normed(st["q"], st["q_w"]), cos, sin))
    k, v = _rotated(_normed(st["k"], st["k_w"]), cos, sin), st["v"].float()
    at, off = st["slots"] // c["page"], st["slots"] % c["page"]
    if st["k_s"] is None:
        st["k_cache"][at, off] = k.to(st["q"].dtype)
        st["v_cache"][at, off] = st["v"]
    else:
        st["k_cache"][at, off], st["k_s"][at, off] = _codes(k)
        st["v_cache"][at, off], st["v_s"][at, off] = _codes(v)
    return [st["q_out"], *_cache_values(st)]


def _attend(q, k, v, seen, scale):
    """q [B, Lq, HQ, D], k / v [B, Lk, HKV, D], seen [B, Lq, Lk]: softmax over the seen keys, zero
    where there are none."""
    b, lq, hq, d = q.shape
    hkv = k.shape[2]
    qh = q.float().reshape(b, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    s = torch.matmul(qh, k.float().permute(0, 2, 3, 1).contiguous()) * scale  # [B, HKV, G * Lq, Lk]
    hide = ~seen[:, None, None]
    s = s.view(b, hkv, hq // hkv, lq, -1).masked_fill_(hide, -math.inf)
    s -= s.amax(-1, keepdim=True).clamp_min_(-3e38)
    p = s.exp_()
    p /= p.sum(-1, keepdim=True).clamp_min_(1e-38)
    o = torch.matmul(p.view(b, hkv, -1, p.shape[-1]), v.float().permute(0, 2, 1, 3).contiguous())
    return o.view(b, hkv, hq // hkv, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d)


def _pages(cache, scale, table):
    """A sequence's keys (or values) next to each other, as numbers: [B, pages * page, HKV, D]."""
    x = cache[table.long()].float()
    if scale is not None:
        x = x * scale[table.long()][..., None]
    return x.flatten(1, 2)


def _padded(cu, n, rows):
    """Rows of a packed tensor by sequence and place, [B, n], and which of them there are."""
    i = torch.arange(n, device="cuda")
    at = cu[:-1, None] + i[None]
    return at.clamp_max(rows - 1).long(), at < cu[1:, None]


def _plain_prompt(st):
    c, q, out = st["case"], st["q"], st["out"]
    rows, there = _padded(st["cu_q"], st["nq"], q.shape[0])
    nq = (st["cu_q"][1:] - st["cu_q"][:-1])[:, None, None]
    if c["kind"] == "prompt":
        k, v, nk = st["k"][rows], st["v"][rows], nq
    else:
        k, v = (_pages(st[x + "_cache"], st[x + "_s"], st["table"]) for x in "kv")
        nk = st["kv_len"][:, None, None]
    i = torch.arange(st["nq"], device="cuda")[None, :, None]
    j = torch.arange(k.shape[1], device="cuda")[None, None, :]
    seen = (j <= i + nk - nq) & (j < nk) & there[:, :, None]
    o = _attend(q[rows], k, v, seen, st["scale"]).to(q.dtype)
    t = torch.arange(q.shape[0], device="cuda")
    b = torch.searchsorted(st["cu_q"][1:].long().contiguous(), t, right=True)
    out.copy_(o[b, t - st["cu_q"].long()[b]])
    return [out]


def _plain_decode(st):
    k, v = (_pages(st[x + "_cache"], st[x + "_s"], st["table"]) for x in "kv")
    seen = torch.arange(k.shape[1], device="cuda")[None, :] < st["kv_len"][:, None]
    st["out"].copy_(_attend(st["q"][:, None], k, v, seen[:, None], st["scale"])[:, 0])
    return [st["out"]]


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "prompt": _plain_prompt, "chunk": _plain_prompt,
            "decode": _plain_decode}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ the same in 64 bits

def _exact_rope(st):
    """Each frequency's pair as a complex number turned by its angle."""
    c, half = st["case"], st["case"]["rot"] // 2
    if c["inter"]:
        axis = [i % 3 if i < 3 * st["sections"][i % 3] else 0 for i in range(half)]
    else:
        axis = [a for a, n in enumerate(st["sections"]) for _ in range(n)]
    turn = torch.stack([st["pos"][a].double() * st["freqs"][i] for i, a in enumerate(axis)], -1)
    turn = torch.polar(torch.ones_like(turn), turn)[:, None, :]

    def turned(x, w):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * (w.double() + 1)
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    def kept(old, scale, new):
        full = old.double() if scale is None else old.double() * scale.double()[..., None]
        if scale is not None:
            step = (new.abs().amax(-1, keepdim=True) / 127).clamp_min(1e-8)
            new = torch.sign(new) * torch.floor(new.abs() / step + 0.5) * step
        full[st["slots"] // c["page"], st["slots"] % c["page"]] = new
        return full

    return [turned(st["q"], st["q_w"]), kept(st["k_cache"], st["k_s"], turned(st["k"], st["k_w"])),
            kept(st["v_cache"], st["v_s"], st["v"].double())]


def _exact_heads(q, k, v, scale, past):
    """One sequence: q [Lq, HQ, D] after `past` earlier keys; k / v [Lk, HKV, D]."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    share = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        kh, vh = k[:, h // share].double(), v[:, h // share].double()
        s = q[:, h].double() @ kh.t() * scale
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(past + 1), -math.inf)
        out[:, h] = torch.softmax(s, -1) @ vh
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(st)
    nq, nk = _lens(case)
    parts, at = [], 0
    for b, (m, n) in enumerate(zip(nq, nk)):
        q = st["q"][at:at + m]
        if n == 0:
            parts.append(torch.zeros(q.shape, dtype=torch.float64, device="cuda"))
        elif case["kind"] == "prompt":
            parts.append(_exact_heads(q, st["k"][at:at + m], st["v"][at:at + m], st["scale"], 0))
        else:
            pages = st["table"][b, :-(-n // case["page"])].long()
            k, v = (st[x][pages].reshape(-1, case["HKV"], case["HD"])[:n] for x in ("k_cache", "v_cache"))
            if st["k_s"] is not None:
                k, v = (x.double() * st[s][pages].reshape(-1, case["HKV"])[:n, :, None]
                        for x, s in ((k, "k_s"), (v, "v_s")))
            parts.append(_exact_heads(q, k, v, st["scale"], n - m))
        at += m
    return [torch.cat(parts)]
