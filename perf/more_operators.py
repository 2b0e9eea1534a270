"""Operators of a decode step of several candidates of one prompt, and how their speed is watched.

The engine answers a prompt with several candidates at once: one prefill, whose keys and
values all candidates read, then steps of one token of each.  The cases are what such a
step does beside the linears and the operators of perf/operators.py:

* shared   attention of one new token of each sequence over a prefix that its group of
           sequences shares, read once for the group, and over its own keys;
* logits   penalties for repeated tokens, biases and a mask of allowed tokens on the
           vocabulary head's rows;
* sample   one token of each row: the k largest logits, cut by probability mass and by
           the share of the largest, drawn by a uniform number; its log probability.

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
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _kernels(name):
    """A module of the package's kernels; the package's directory is no Python identifier, so it
    is loaded under an alias."""
    if ALIAS not in sys.modules:
        pkg = ROOT / "qwen_3.5_comfy_prompt_enhancer_amd"
        spec = importlib.util.spec_from_file_location(ALIAS, pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[ALIAS] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module(f"{ALIAS}.kernels.{name}")


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # the smallest step: four candidates of a short prompt, early in their answers
        dict(name="shared-4x180", kind="shared", G=1, N=4, L=180, own=40, even=False, pad=0, mix=1, HQ=8, HKV=2,
             HD=256, dt="bf16", kv="16", page=64),
        # the engine's most candidates of the longest prompt it takes
        dict(name="shared-8x8000", kind="shared", G=1, N=8, L=8000, own=190, even=False, pad=0, mix=2, HQ=8, HKV=2,
             HD=256, dt="bf16", kv="16", page=64),
        # the same over a very long prompt in int8, well into the answers
        dict(name="shared-8x100003-int8", kind="shared", G=1, N=8, L=100003, own=700, even=False, pad=0, mix=3, HQ=8,
             HKV=2, HD=256, dt="bf16", kv="int8", page=64),
        # six prompts of different lengths with up to eight candidates each, in a batch padded by three
        # rows; fp16, three query heads to a key head, small pages
        dict(name="shared-6-prompts", kind="shared", G=6, N=8, L=6000, own=300, even=False, pad=3, mix=4, HQ=12,
             HKV=4, HD=128, dt="fp16", kv="16", page=16),
        # a full serving batch behind one long instruction, eight query heads to a key head
        dict(name="shared-64x16384", kind="shared", G=1, N=64, L=16384, own=1000, even=False, pad=0, mix=5, HQ=32,
             HKV=4, HD=128, dt="fp16", kv="16", page=32),
        # one row of the vocabulary head with the penalties of a short answer
        dict(name="logits-1", kind="logits", B=1, V=248320, L=600, prompt=400, bias=0, mask=False, even=True, mix=0,
             dt="bf16", to="fp32"),
        # eight candidates under a grammar, with a user's biases
        dict(name="logits-8-grammar", kind="logits", B=8, V=248320, L=1500, prompt=1000, bias=40, mask=True, even=False,
             mix=6, dt="bf16", to="fp32"),
        # a vocabulary of odd size, results in 16 bits
        dict(name="logits-5x50021", kind="logits", B=5, V=50021, L=37, prompt=20, bias=3, mask=True, even=False,
             mix=7, dt="fp16", to="fp16"),
        # a full serving batch with long histories
        dict(name="logits-64", kind="logits", B=64, V=248320, L=8192, prompt=7000, bias=300, mask=True, even=False,
             mix=8, dt="bf16", to="fp32"),
        # one token of one sequence
        dict(name="sample-1", kind="sample", B=1, V=248320, k=20, masked=False, dt="fp32"),
        # the vocabulary head's own 16-bit rows (many of equal value), an odd vocabulary
        dict(name="sample-5x50021-bf16", kind="sample", B=5, V=50021, k=64, masked=False, dt="bf16"),
        # a full serving batch, some rows under grammars
        dict(name="sample-64", kind="sample", B=64, V=248320, k=50, masked=True, dt="fp32"),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "logits", "sample"])
    mix = rng.randrange(1, 1 << 20)
    if kind == "shared":
        hkv = rng.choice([1, 2, 4, 5])
        hq, hd = hkv * rng.choice([1, 3, 4, 4, 8]), rng.choice([64, 128, 256, 256])
        g = _log(rng, 1, 8)
        n = _log(rng, 1, 64 // g)
        # pairs of a query and a prefix key, and cache bytes, at most what the largest listed case has
        most = min(64 * 32 * 128 * 16384 // (g * n * hq * hd), 100003 * 512 // (g * hkv * hd), 131072)
        return dict(kind=kind, G=g, N=n, L=_log(rng, 1, most), own=_log(rng, 1, min(4096, 32_000_000 // (g * n * hkv * hd))),
                    even=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 5]), mix=mix, HQ=hq, HKV=hkv, HD=hd,
                    dt=rng.choice(["bf16", "bf16", "fp16"]), kv=rng.choice(["16", "16", "int8"]),
                    page=rng.choice([16, 32, 64, 128]))
    v = _log(rng, 500, 262144)
    b = _log(rng, 1, min(64, 64 * 248320 // v))
    dt = rng.choice(["bf16", "fp16", "fp32"])
    if kind == "logits":
        n = _log(rng, 1, 8192)
        return dict(kind=kind, B=b, V=v, L=n, prompt=rng.randint(0, n), bias=rng.choice([0, 1, 17, 300]),
                    mask=rng.random() < 0.6, even=rng.random() < 0.3, mix=mix, dt=dt, to=rng.choice(["fp32", "fp32", dt]))
    return dict(kind=kind, B=b, V=v, k=_log(rng, 1, 128), masked=rng.random() < 0.5, dt=dt)


def _shares(case):
    """Sequences of each group, prefix keys of each group, own keys of each sequence.  Uneven
    batches: the first of each is the longest; with three groups and more the second prefix is
    empty, with five and more the fourth group is (a padded entry)."""
    g, n, rng = case["G"], case["N"], random.Random(case["mix"])
    if case["even"]:
        return [n] * g, [case["L"]] * g, [case["own"]] * (g * n)
    size = [n if i == 0 else rng.randint(1, n) for i in range(g)]
    pre = [case["L"] if i == 0 else rng.randint(1, case["L"]) for i in range(g)]
    if g > 2:
        pre[1] = 0
    if g > 4:
        size[3] = 0
    return size, pre, [case["own"] if i == 0 else rng.randint(1, case["own"]) for i in range(sum(size))]


def _histories(case):
    """(tokens, of them the prompt's) of each row."""
    rng = random.Random(case["mix"])
    n = [case["L"] if i == 0 or case["even"] else rng.randint(0, case["L"]) for i in range(case["B"])]
    return n, [min(x, case["prompt"]) for x in n]


def work(case):
    if case["kind"] == "shared":
        size, pre, mine = _shares(case)
        hq, hkv, hd = case["HQ"], case["HKV"], case["HD"]
        kvb = hd * 2 if case["kv"] == "16" else hd + 4                # bytes of a token's key of one head
        keys = sum(p for p, n in zip(pre, size) if n) + sum(mine)
        pairs = sum(p * n for p, n in zip(pre, size)) + sum(mine)
        rows = 4 * sum(-(-n // case["page"]) for n in pre + mine) + 4 * (2 * len(pre) + 1 + len(mine))
        return {"bytes": 2 * len(mine) * hq * hd * 2 + 2 * keys * hkv * kvb + rows, "flops": 4 * pairs * hq * hd}
    b, v = case["B"], case["V"]
    if case["kind"] == "logits":
        n, _ = _histories(case)
        read = b * v * BYTES[case["dt"]] + 4 * sum(n) + 20 * b + 8 * b * case["bias"] + case["mask"] * 4 * b * -(-v // 32)
        return {"bytes": read + b * v * BYTES[case["to"]], "flops": b * v + 6 * sum(n) + b * case["bias"]}
    return {"bytes": b * v * BYTES[case["dt"]] + 28 * b, "flops": 4 * b * v}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1 + seed)


def _randn(g, shape, dt):
    return torch.randn(shape, generator=g, device="cuda").to(dt)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


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


def _tables(order, page, *lens):
    """A page table for each list of lengths, pages taken from `order` in turn."""
    at, out = 0, []
    for ns in lens:
        need = [-(-n // page) for n in ns]
        t = torch.zeros((len(ns), max(1, *need)), dtype=torch.int32)
        for b, n in enumerate(need):
            t[b, :n] = order[at:at + n]
            at += n
        out.append(t.cuda())
    return out


def _logit_rows(g, case):
    """Rows of the vocabulary head: a flat bulk, and a few hundred tokens that stand out."""
    b, v = case["B"], case["V"]
    x = torch.randn((b, v), generator=g, device="cuda") * 2
    some = torch.rand((b, v), generator=g, device="cuda") < 300 / v
    return torch.where(some, torch.randn((b, v), generator=g, device="cuda") * 2.5 + 10, x)


def _prepare_shared(case, g):
    size, pre, mine = _shares(case)
    dt, hq, hd, rows = DTYPES[case["dt"]], case["HQ"], case["HD"], len(mine) + case["pad"]
    mine_padded = mine + [0] * case["pad"]
    pages = sum(-(-n // case["page"]) for n in pre + mine) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    prefix_table, table = _tables(order, case["page"], pre, mine_padded)
    at = [sum(size[:i]) for i in range(len(size) + 1)]
    return dict(scale=hd ** -0.5, q=_randn(g, (rows, hq, hd), dt) * 2, out=torch.zeros((rows, hq, hd), dtype=dt, device="cuda"),
                prefix_table=prefix_table, prefix_len=_ints(pre), cu_seq=_ints(at), table=table,
                kv_len=_ints(mine_padded), n=max(size), **_cache(g, case, pages))


def _prepare_logits(case, g):
    b, v, (n, p) = case["B"], case["V"], _histories(case)
    x = _logit_rows(g, case)
    # histories repeat themselves, and hold many of the tokens that stand out
    tokens = (torch.rand((b, case["L"]), generator=g, device="cuda") ** 3 * v).to(torch.int64)
    top = x.topk(min(v, 64), 1).indices
    pick = torch.randint(0, top.shape[1], tokens.shape, generator=g, device="cuda")
    often = torch.rand(tokens.shape, generator=g, device="cuda") < 0.2
    tokens = torch.where(often, top.gather(1, pick), tokens).to(torch.int32)
    st = dict(logits=x.to(DTYPES[case["dt"]]), out=torch.empty((b, v), dtype=DTYPES[case["to"]], device="cuda"),
              tokens=tokens, lens=_ints(n), prompt_lens=_ints(p), bias_ids=None, bias=None, mask=None,
              repetition=1 + torch.rand(b, generator=g, device="cuda") * 0.3,
              presence=torch.rand(b, generator=g, device="cuda") * 1.5,
              frequency=torch.rand(b, generator=g, device="cuda") * 0.5)
    if case["bias"]:
        m = min(case["bias"], v)
        # ids of a row differ
        st["bias_ids"] = torch.rand((b, v), generator=g, device="cuda").topk(m, 1).indices.to(torch.int32)
        st["bias"] = torch.randn((b, m), generator=g, device="cuda") * 5
    if case["mask"]:
        st["mask"] = torch.randint(-2 ** 31, 2 ** 31, (b, -(-v // 32)), generator=g, device="cuda").to(torch.int32)
    return st


def _prepare_sample(case, g):
    b, v = case["B"], case["V"]
    x = _logit_rows(g, case)
    if case["masked"]:
        # every second row allows a few tokens in a hundred, one row in eight fewer than k
        share = torch.tensor([1.0, 0.03, 1.0, 0.03, 1.0, 0.03, 1.0, 2.0 / v], device="cuda")[torch.arange(b, device="cuda") % 8]
        hide = torch.rand((b, v), generator=g, device="cuda") >= share[:, None]
        hide.scatter_(1, torch.randint(0, v, (b, 1), generator=g, device="cuda"), False)
        x = x.masked_fill(hide, -math.inf)
    return dict(logits=x.to(DTYPES[case["dt"]]), u=torch.rand(b, generator=g, device="cuda"), k=min(case["k"], v),
                tokens=torch.empty(b, dtype=torch.int64, device="cuda"), logprobs=torch.empty(b, device="cuda"),
                temperature=torch.rand(b, generator=g, device="cuda") + 0.3,
                top_p=torch.rand(b, generator=g, device="cuda") * 0.4 + 0.6,
                min_p=torch.rand(b, generator=g, device="cuda") * 0.05)


def prepare(case, seed):
    make = {"shared": _prepare_shared, "logits": _prepare_logits, "sample": _prepare_sample}[case["kind"]]
    return dict(case=case, **make(case, _gen(seed)))


# ------------------------------------------------------------------ one pass

def _own(st):
    kind = st["case"]["kind"]
    if kind == "shared":
        _kernels("attention").attn_decode_shared(
            st["q"], st["k_cache"], st["v_cache"], st["prefix_table"], st["prefix_len"], st["cu_seq"], st["table"],
            st["kv_len"], st["out"], k_s=st["k_s"], v_s=st["v_s"], scale=st["scale"])
        return [st["out"]]
    if kind == "logits":
        _kernels("sampling").logits_process(
            st["logits"], st["out"], tokens=st["tokens"], lens=st["lens"], prompt_lens=st["prompt_lens"],
            repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"], bias_ids=st["bias_ids"],
            bias=st["bias"], mask=st["mask"])
        return [st["out"]]
    _kernels("sampling").sample(st["logits"], st["u"], st["tokens"], logprobs=st["logprobs"], top_k=st["k"],
                                temperature=st["temperature"], top_p=st["top_p"], min_p=st["min_p"])
    return [st["tokens"], st["logprobs"]]


def _pages(cache, scale, table):
    """The keys (or values) of each row of a table next to each other, as numbers: [rows, pages * page, HKV, D]."""
    x = cache[table.long()].float()
    if scale is not None:
        x = x * scale[table.long()][..., None]
    return x.flatten(1, 2)


def _part(q, k, v, n, scale):
    """q [S, HKV, R, D] over the first n [S] of k / v [S, Lk, HKV, D]: maximum, sum and values of the
    softmax, not yet divided."""
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * scale            # [S, HKV, R, Lk]
    hide = torch.arange(k.shape[1], device="cuda")[None, :] >= n[:, None]
    s = s.masked_fill_(hide[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min_(-3e38)
    p = (s - m).exp_()
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())


def _plain_shared(st):
    c, q, out = st["case"], st["q"], st["out"]
    (b, hq, d), hkv, n = q.shape, c["HKV"], st["n"]
    share, cu = hq // hkv, st["cu_seq"].long()
    qh = q.float().view(b, hkv, share, d)
    # the prefix: a group's sequences as rows of one product
    at = (cu[:-1, None] + torch.arange(n, device="cuda")).clamp_max(b - 1)     # [G, N]
    qg = qh[at].permute(0, 2, 1, 3, 4).reshape(c["G"], hkv, n * share, d)
    pm, pl, po = (x.view(c["G"], hkv, n, share, -1).transpose(1, 2) for x in _part(
        qg, *(_pages(st[x + "_cache"], st[x + "_s"], st["prefix_table"]) for x in "kv"), st["prefix_len"], st["scale"]))
    om, ol, oo = _part(qh, *(_pages(st[x + "_cache"], st[x + "_s"], st["table"]) for x in "kv"), st["kv_len"], st["scale"])
    # both parts of each sequence
    i = torch.arange(b, device="cuda")
    g = torch.searchsorted(cu[1:].contiguous(), i, right=True).clamp_max(c["G"] - 1)
    place = (i - cu[g]).clamp_max(n - 1)
    pm, pl, po = pm[g, place], pl[g, place], po[g, place]
    m = torch.maximum(pm, om)
    ep, eo = (pm - m).exp(), (om - m).exp()
    o = (po * ep + oo * eo) / (pl * ep + ol * eo).clamp_min(1e-38)
    out.copy_(torch.where((i < cu[-1])[:, None, None], o.view(b, hq, d), out.float()))
    return [out]


def _plain_logits(st):
    x = st["logits"].float()
    b, v = x.shape
    i = torch.arange(st["tokens"].shape[1], device="cuda")
    there, answer = i < st["lens"][:, None], i >= st["prompt_lens"][:, None]
    ids = st["tokens"].long()
    seen = torch.zeros((b, v + 1), dtype=torch.bool, device="cuda").scatter_(1, torch.where(there, ids, v), True)[:, :v]
    count = torch.zeros((b, v + 1), dtype=torch.int32, device="cuda")
    count = count.scatter_add_(1, torch.where(there & answer, ids, v), torch.ones_like(st["tokens"]))[:, :v]
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    if st["bias"] is not None:
        x = x.scatter_add(1, st["bias_ids"].long(), st["bias"])
    if st["mask"] is not None:
        bits = (st["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x = x.masked_fill(bits.flatten(1)[:, :v] == 0, -math.inf)
    st["out"].copy_(x)
    return [st["out"]]


def _plain_sample(st):
    x = st["logits"].float()
    b, v = x.shape
    # largest first, of equal ones the first: an order-preserving integer of the value, then the place
    bits = torch.where(x == 0, 0.0, x).view(torch.int32).long()
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) | (v - 1 - torch.arange(v, device="cuda"))
    ids = v - 1 - (key.topk(st["k"], 1).values & 0xFFFFFFFF)
    y = x.gather(1, ids).double()
    top = y[:, :1]
    w = torch.where(y == top, 1.0, ((y - top) / st["temperature"].double()[:, None]).exp())
    cum = w.cumsum(1)
    keep = ((cum - w) < st["top_p"].double()[:, None] * cum[:, -1:]) & (w >= st["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    cum = w.cumsum(1)
    at = (cum <= st["u"].double()[:, None] * cum[:, -1:]).sum(1).clamp_max(st["k"] - 1)
    st["tokens"].copy_(ids.gather(1, at[:, None])[:, 0])
    m = x.amax(1)
    total = (x - m[:, None]).exp().sum(1, dtype=torch.float64)
    st["logprobs"].copy_(y.gather(1, at[:, None])[:, 0] - m - total.log())
    return [st["tokens"], st["logprobs"]]


def run(state):
    if own:
        return _own(state)
    return {"shared": _plain_shared, "logits": _plain_logits, "sample": _plain_sample}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ the same in 64 bits

def _exact_shared(st):
    """Sequence by sequence, over its prefix and its own keys in a row."""
    c = st["case"]
    size, pre, mine = _shares(c)
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    share = c["HQ"] // c["HKV"]

    def keys(table, n):
        ids = table[:-(-n // c["page"])].long()
        got = []
        for x, s in (("k_cache", "k_s"), ("v_cache", "v_s")):
            y = st[x][ids].reshape(-1, c["HKV"], c["HD"])[:n].double()
            if st[s] is not None:
                y = y * st[s][ids].reshape(-1, c["HKV"])[:n, :, None].double()
            got.append(y)
        return got

    b = 0
    for g, n in enumerate(size):
        kp, vp = keys(st["prefix_table"][g], pre[g])
        for _ in range(n):
            ko, vo = keys(st["table"][b], mine[b])
            for h in range(c["HKV"]):
                k, v = torch.cat([kp[:, h], ko[:, h]]), torch.cat([vp[:, h], vo[:, h]])
                q = st["q"][b, h * share:(h + 1) * share].double()
                out[b, h * share:(h + 1) * share] = torch.softmax(q @ k.t() * st["scale"], -1) @ v
            b += 1
    return [out]


def _exact_logits(st):
    """Row by row, with the history's distinct tokens and how often each came."""
    n, p = _histories(st["case"])
    v, rows = st["case"]["V"], []
    for b, x in enumerate(st["logits"].double()):
        ids = torch.unique(st["tokens"][b, :n[b]]).long()
        x[ids] = torch.where(x[ids] > 0, x[ids] / st["repetition"][b].double(), x[ids] * st["repetition"][b].double())
        ids, times = torch.unique(st["tokens"][b, p[b]:n[b]], return_counts=True)
        x[ids.long()] -= st["frequency"][b].double() * times + st["presence"][b].double()
        if st["bias"] is not None:
            x[st["bias_ids"][b].long()] += st["bias"][b].double()
        if st["mask"] is not None:
            i = torch.arange(v, device="cuda")
            word = st["mask"][b].long()[i // 32] & 0xFFFFFFFF
            x[(word // 2 ** (i % 32)) % 2 == 0] = -math.inf
        rows.append(x)
    return [torch.stack(rows)]


def _exact_sample(st):
    """Row by row: the sorted row's first k, weights kept one after the other, the draw."""
    tokens, logs = [], []
    for b, x in enumerate(st["logits"].double()):
        val, ids = torch.sort(x, descending=True, stable=True)
        y = val[:st["k"]].tolist()
        t, top_p, min_p, u = (float(st[n][b]) for n in ("temperature", "top_p", "min_p", "u"))
        w = [math.exp((z - y[0]) / t) for z in y]
        kept, before = [], 0.0
        for z in w:
            kept.append(z if not kept or (before < top_p * math.fsum(w) and z >= min_p) else 0.0)
            before += z
        goal, at, run_sum = u * math.fsum(kept), 0, kept[0]
        while run_sum <= goal and at + 1 < len(kept):
            at += 1
            run_sum += kept[at]
        tokens.append(int(ids[at]))
        logs.append(y[at] - float(torch.logsumexp(x, 0)))
    return [torch.tensor(tokens, device="cuda"), torch.tensor(logs, dtype=torch.float64, device="cuda")]


def exact(case, seed):
    st = prepare(case, seed)
    return {"shared": _exact_shared, "logits": _exact_logits, "sample": _exact_sample}[case["kind"]](st)
