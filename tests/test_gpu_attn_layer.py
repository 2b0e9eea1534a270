"""The attention operators as an engine uses them: together, with the projections around them,
captured, on several streams, over caches past 4 GiB, and with contents that name no page."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R
import helpers as H

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
HQ, HKV, HD, HID = 8, 2, 256, 2048


def _freqs(half=32):
    return torch.tensor([1e7 ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")


class Layer:
    """One attention layer's mixer with its projections (engine.py:244-268): RMSNorm + proj3,
    qk_norm_rope into the cache, attention, gates, output projection into the residual."""

    def __init__(self, rows, int8, seed=0, pages=40, page=16):
        from qwen35_amd.kernels import attention, gemm, norm
        self.A, self.G, self.N = attention, gemm, norm
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w = [tuple(x.cuda() for x in H.engine_w8(HID, n, seed + i)) for i, n in
                  enumerate((2 * HQ * HD, HKV * HD, HKV * HD))]
        self.wo = tuple(x.cuda() for x in H.engine_w8(HQ * HD, HID, seed + 5))
        self.nw = (torch.randn(HID, generator=g, device="cuda") * 0.1).to(BF)
        self.qw, self.kw = ((torch.randn(HD, generator=g, device="cuda") * 0.2).to(BF) for _ in range(2))
        self.cache = R.cache(pages, page, HKV, HD, BF, seed + 7, int8)
        self.freqs = _freqs()
        self.proj = torch.empty((rows, 2 * HQ * HD + 2 * HKV * HD), dtype=BF, device="cuda")
        self.q = torch.empty((rows, HQ, HD), dtype=BF, device="cuda")
        self.out = torch.empty((rows, HQ, HD), dtype=BF, device="cuda")
        self.codes = torch.empty((rows, HID), dtype=torch.int8, device="cuda")
        self.scales = torch.empty((rows, HID // 64), dtype=torch.float32, device="cuda")

    def run(self, hidden, pos, slots, attend):
        n = hidden.shape[0]
        proj, q, out, codes, scales = (x[:n] for x in (self.proj, self.q, self.out, self.codes, self.scales))
        self.N.rmsnorm_quant(hidden, self.nw, codes, scales)
        self.G.proj3(codes, scales, *self.w[0], *self.w[1], *self.w[2], proj)
        kc, vc, ks, vs = self.cache
        k0 = 2 * HQ * HD
        self.A.qk_norm_rope(proj[:, :k0].view(n, HQ, 2 * HD)[..., :HD], proj[:, k0:k0 + HKV * HD].view(n, HKV, HD), pos,
                            self.freqs, q, v=proj[:, k0 + HKV * HD:].view(n, HKV, HD), k_cache=kc, v_cache=vc,
                            slots=slots, k_s=ks, v_s=vs, q_w=self.qw, k_w=self.kw, sections=[12, 10, 10],
                            interleaved=True)
        attend(q, out)
        self.N.gate_mul_quant(out.view(n, HQ * HD), proj[:, :k0], codes, scales, hd=HD)
        self.G.gemm_i8(codes, scales, *self.wo, hidden, residual=hidden)

    def paged(self, table, kv_len, cu):
        kc, vc, ks, vs = self.cache
        return lambda q, out: self.A.attn_prompt_paged(q, kc, vc, table, kv_len, cu, out, k_s=ks, v_s=vs)

    def decode(self, table, kv_len):
        kc, vc, ks, vs = self.cache
        return lambda q, out: self.A.attn_decode(q, kc, vc, table, kv_len, out, k_s=ks, v_s=vs)


def _ints(x, dt=torch.int32):
    return torch.tensor(x, dtype=dt, device="cuda")


def _slots(table, b, first, n, page):
    i = torch.arange(first, first + n, device="cuda")
    return table[b, i // page].long() * page + i % page


@pytest.mark.parametrize("int8", [False, True])
def test_a_prompt_in_chunks_and_tokens_after_it(int8):
    """Two sequences' prompts in two chunks each, then three tokens: every step's attention equals
    attention in 64 bits over the rotated queries of that step and what the cache then holds, and
    the cache holds the keys of all steps."""
    page, L = 16, Layer(64, int8, seed=int(int8))
    lens, done = [75, 31], [0, 0]
    table, _ = R.pages_of([n + 8 for n in lens], page, 0, 3, "cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    steps = [[40, 17], [35, 14], [1, 1], [1, 1], [1, 1]]
    for step in steps:
        n = sum(step)
        hidden = torch.randn((n, HID), generator=g, device="cuda").to(BF)
        before = hidden.clone()
        at = torch.cat([torch.arange(d, d + m, device="cuda") for d, m in zip(done, step)])
        pos = torch.stack([at, at // 3, at % 7])
        slots = torch.cat([_slots(table, b, d, m, page) for b, (d, m) in enumerate(zip(done, step))])
        done = [d + m for d, m in zip(done, step)]
        kv = _ints(done)
        L.run(hidden, pos, slots, L.decode(table, kv) if n == 2 else L.paged(table, kv, _ints([0, step[0], n])))
        torch.cuda.synchronize()
        row = 0
        for b, m in enumerate(step):
            k, v = R.gathered(L.cache, table, b, done[b])
            ref, tol = R.attend(L.q[row:row + m], k, v, HD ** -0.5, R.causal(m, done[b], "cuda"), BF)
            R.check(L.out[row:row + m], ref, tol, f"step {step} sequence {b}")
            row += m
        assert torch.isfinite(hidden.float()).all() and not torch.equal(hidden, before)
    # the keys of all steps are where the table says, in order: rotated by their own positions
    k0 = 2 * HQ * HD
    x = L.proj[1:2, k0:k0 + HKV * HD].view(1, HKV, HD).double()     # the last token of the second sequence
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (L.kw.double() + 1)
    p = done[1] - 1
    axis = [i % 3 if i < 3 * [12, 10, 10][i % 3] else 0 for i in range(32)]
    ang = torch.tensor([[p, p // 3, p % 7][a] for a in axis], dtype=torch.float64, device="cuda") * L.freqs
    a, c = y[..., :32], y[..., 32:64]
    want = torch.cat([a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin(), y[..., 64:]], -1)[0]
    got = R.gathered(L.cache, table, 1, done[1])[0][-1]
    step = want.abs().amax(-1, keepdim=True) / 127 * 0.51 if int8 else want.abs() * 2.0 ** -8
    assert ((got - want).abs() <= step + 1e-4 * want.abs().amax()).all()


def test_a_chunked_prompt_agrees_with_the_whole_one():
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(1)
    n, page = 300, 32
    q, k, v = (torch.randn((n, h, HD), generator=g, device="cuda").to(BF) for h in (HQ, HKV, HKV))
    table, pages = R.pages_of([n], page, 2, 4, "cuda")
    c = R.cache(pages, page, HKV, HD, BF, 2)
    s = _slots(table, 0, 0, n, page)
    c[0][s // page, s % page], c[1][s // page, s % page] = k, v
    whole = torch.empty_like(q)
    A.attn_prompt(q, k, v, _ints([0, n]), whole)
    parts = torch.empty_like(q)
    for a, b in ((0, 130), (130, 131), (131, 300)):
        A.attn_prompt_paged(q[a:b], c[0], c[1], table, _ints([b]), _ints([0, b - a]), parts[a:b])
    one = torch.empty((1, HQ, HD), dtype=BF, device="cuda")
    A.attn_decode(q[n - 1:], c[0], c[1], table, _ints([n]), one)
    ref, tol = R.attend(q, k, v, HD ** -0.5, R.causal(n, n, "cuda"), BF)
    for y, r in ((whole, slice(0, n)), (parts, slice(0, n)), (one, slice(n - 1, n))):
        R.check(y, ref[r], tol[r])


def test_a_captured_decode_step_replays():
    """One graph of a whole decode step; lengths, positions and slots change in place between
    replays, with eager work and synchronizations between them; every replay equals the eager step
    bit for bit."""
    from qwen35_amd.kernels import qlin as C
    page, B = 16, 3
    lens = [500, 3, 64]
    table, pages = R.pages_of([n + 16 for n in lens], page, 2, 6, "cuda")
    L, E = (Layer(B, False, seed=2, pages=pages, page=page) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(7)
    hidden = torch.zeros((B, HID), dtype=BF, device="cuda")
    pos, slots, kv = (_ints([0] * B, dt) for dt in (torch.int64, torch.int64, torch.int32))
    pos3 = pos[None].expand(3, B).contiguous()

    def step(M):
        M.run(hidden, pos3, slots, M.decode(table, kv))

    def prepare(t):
        at = torch.tensor([n + t for n in lens], device="cuda")
        pos3.copy_(torch.stack([at, at // 2, at % 5]))
        slots.copy_(table[torch.arange(B, device="cuda"), at // page].long() * page + at % page)
        kv.copy_(at + 1)
        hidden.copy_(torch.randn((B, HID), generator=g, device="cuda"))

    prepare(0)
    step(L)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        step(L)
    L.cache[0].copy_(E.cache[0])
    L.cache[1].copy_(E.cache[1])
    for t in range(6):
        prepare(t)
        h0 = hidden.clone()
        graph.replay()
        if t % 2:
            torch.cuda.synchronize()
        got = hidden.clone()
        hidden.copy_(h0)
        step(E)
        torch.cuda.synchronize()
        assert torch.equal(got, hidden) and torch.equal(L.out, E.out), t
        assert torch.equal(L.cache[0], E.cache[0]) and torch.equal(L.cache[1], E.cache[1]), t


@pytest.mark.parametrize("hd,T,bounds", [
    (256, 3333, [[0, 3333, 3333], [0, 1, 3000], [0, 1700, 3333], [0, 0, 0], [0, 3333, 3333]]),  # joined by a launch
    (256, 6000, [[0, 5900, 6000], [0, 3000, 6000], [0, 17, 33], [0, 5900, 6000]]),                # by the last part
    (64, 700, [[0, 700, 700], [0, 350, 700], [0, 699, 700]]),                                     # halved tiles
])
def test_a_captured_prompt_replays_with_other_bounds(hd, T, bounds):
    """Cuts and joins follow the bounds that the device holds: every replay equals the eager call bit
    for bit, and rows of no sequence stay as they were."""
    from qwen35_amd.kernels import attention as A, qlin as C
    g = torch.Generator(device="cuda").manual_seed(T)
    q, k, v = (torch.randn((T, h, hd), generator=g, device="cuda").to(BF) for h in (8, 2, 2))
    out, want, cu = torch.empty_like(q), torch.empty_like(q), _ints(bounds[0])
    A.attn_prompt(q, k, v, cu, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        A.attn_prompt(q, k, v, cu, out)
    for n, b in enumerate(bounds):
        cu.copy_(_ints(b))
        out.fill_(7)
        want.fill_(7)
        graph.replay()
        if n % 2:
            torch.cuda.synchronize()
        A.attn_prompt(q, k, v, cu, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want), b
        assert (out[b[-1]:] == 7).all()
        one = b[1]
        if one:  # the first sequence by itself
            ref, tol = R.attend(q[one - 1:one], k[:one], v[:one], hd ** -0.5,
                                torch.ones((1, one), dtype=torch.bool, device="cuda"), BF)
            R.check(out[one - 1:one], ref, tol, f"bounds {b}")


def test_two_graphs_of_one_stream_share_its_workspace():
    """A decode call and a prompt call cut into parts, captured apart and replayed in turn."""
    from qwen35_amd.kernels import attention as A, qlin as C
    g = torch.Generator(device="cuda").manual_seed(9)
    q = torch.randn((900, HQ, HD), generator=g, device="cuda").to(BF)
    k, v = (torch.randn((900, HKV, HD), generator=g, device="cuda").to(BF) for _ in range(2))
    table, pages = R.pages_of([9000], 64, 1, 4, "cuda")
    c = R.cache(pages, 64, HKV, HD, BF, 2)
    n, cu = _ints([9000]), _ints([0, 900])
    o1, o2 = torch.empty_like(q), torch.empty_like(q[:1])
    runs = [lambda: A.attn_prompt(q, k, v, cu, o1), lambda: A.attn_decode(q[:1], c[0], c[1], table, n, o2)]
    want = []
    for r, o in zip(runs, (o1, o2)):
        r()
        want.append(o.clone())
    graphs = []
    for r in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with C.capture(graphs[-1]):
            r()
    for _ in range(4):
        for o in (o1, o2):
            o.zero_()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, want[0]) and torch.equal(o2, want[1])


def test_streams_run_side_by_side():
    """The same calls on two streams at once, each with the workspace of its own."""
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(10)
    table, pages = R.pages_of([7000, 3000], 64, 1, 4, "cuda")
    c = R.cache(pages, 64, HKV, HD, BF, 2)
    q = torch.randn((600, HQ, HD), generator=g, device="cuda").to(BF)
    kv, cu = _ints([7000, 3000]), _ints([0, 200, 600])
    want = [torch.empty_like(q), torch.empty_like(q[:2])]
    A.attn_prompt_paged(q, c[0], c[1], table, kv, cu, want[0])
    A.attn_decode(q[:2], c[0], c[1], table, kv, want[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(2)], [torch.empty_like(q[:2]) for _ in range(2)]]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                A.attn_prompt_paged(q, c[0], c[1], table, kv, cu, outs[0][i])
                A.attn_decode(q[:2], c[0], c[1], table, kv, outs[1][i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[0][i], want[0]) and torch.equal(outs[1][i], want[1])


def test_linears_on_the_same_workspace_are_what_they_were():
    """The split linears' counters and the attention calls' are the same memory."""
    from qwen35_amd.kernels import attention as A, gemm
    a, a_s = (x.cuda() for x in H.engine_act(64, 2048, 1))
    b, b_s = (x.cuda() for x in H.engine_w8(2048, 2048, 2))
    outs = [torch.empty((64, 2048), dtype=BF, device="cuda") for _ in range(2)]
    gemm.gemm_i8(a, a_s, b, b_s, outs[0])
    g = torch.Generator(device="cuda").manual_seed(11)
    q = torch.randn((1000, HQ, HD), generator=g, device="cuda").to(BF)
    k, v = (torch.randn((1000, HKV, HD), generator=g, device="cuda").to(BF) for _ in range(2))
    o = torch.empty_like(q)
    for _ in range(3):
        A.attn_prompt(q, k, v, _ints([0, 1000]), o)
        gemm.gemm_i8(a, a_s, b, b_s, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(*outs)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 elements: the last pages hold the sequence."""
    from qwen35_amd.kernels import attention as A
    page, hkv, hd = 64, 4, 256
    per = page * hkv * hd
    pages = (1 << 32) // per + 40
    for int8 in (False, True):
        dt = torch.int8 if int8 else BF
        k, v = (torch.empty((pages, hkv, page, hd), dtype=dt, device="cuda").transpose(1, 2) for _ in range(2))
        ks, vs = ((torch.full((pages, hkv, page), 0.01, device="cuda").transpose(1, 2)) if int8 else None for _ in range(2))
        n = 16 * page - 5
        table = torch.arange(pages - 16, pages, dtype=torch.int32, device="cuda")[None]
        for x in (k, v):
            fresh = torch.randn((16, page, hkv, hd), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
            x[pages - 16:] = (fresh * 30).to(torch.int8) if int8 else fresh.to(BF)
        g = torch.Generator(device="cuda").manual_seed(4)
        q = torch.randn((40, 8, hd), generator=g, device="cuda").to(BF)
        # the last 40 tokens' keys and values come by way of qk_norm_rope
        new = torch.randn((40, 2 * hkv * hd), generator=g, device="cuda").to(BF)
        i = torch.arange(n - 40, n, device="cuda")
        slots = table[0, i // page].long() * page + i % page
        qr = torch.empty_like(q)
        A.qk_norm_rope(q, new[:, :hkv * hd].view(40, hkv, hd), i, _freqs(), qr, v=new[:, hkv * hd:].view(40, hkv, hd),
                       k_cache=k, v_cache=v, slots=slots, k_s=ks, v_s=vs)
        o, o1 = torch.empty_like(q), torch.empty_like(q[:1])
        A.attn_prompt_paged(qr, k, v, table, _ints([n]), _ints([0, 40]), o, k_s=ks, v_s=vs)
        A.attn_decode(qr[39:], k, v, table, _ints([n]), o1, k_s=ks, v_s=vs)
        torch.cuda.synchronize()
        kk, vv = R.gathered((k, v, ks, vs), table, 0, n)
        assert torch.equal(vv[-1].to(BF), new[39, hkv * hd:].view(hkv, hd)) or int8
        ref, tol = R.attend(qr, kk, vv, hd ** -0.5, R.causal(40, n, "cuda"), BF)
        R.check(o, ref, tol, "prompt")
        R.check(o1, ref[39:], tol[39:], "decode")
        del k, v, ks, vs
        torch.cuda.empty_cache()


@pytest.mark.parametrize("int8", [False, True])
def test_contents_that_name_no_page_or_too_many_keys(int8):
    """A sequence with a page outside the cache is NaN, whichever of its keys lie there; the others
    are what they were.  Lengths count as what the table can hold; row bounds as the rows there are."""
    from qwen35_amd.kernels import attention as A
    page, lens = 16, [200, 333, 64]
    table, pages = R.pages_of(lens, page, 2, 8, "cuda")
    c = R.cache(pages, page, HKV, HD, BF, 3, int8)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn((3, HQ, HD), generator=g, device="cuda").to(BF)
    qp = torch.randn((90, HQ, HD), generator=g, device="cuda").to(BF)
    kv, cu = _ints(lens), _ints([0, 40, 60, 90])

    def both(table, kv, cu):
        o, op = torch.full_like(q, 7.0), torch.full_like(qp, 7.0)
        A.attn_decode(q, c[0], c[1], table, kv, o, k_s=c[2], v_s=c[3])
        A.attn_prompt_paged(qp, c[0], c[1], table, kv, cu, op, k_s=c[2], v_s=c[3])
        torch.cuda.synchronize()
        return o, op

    o, op = both(table, kv, cu)
    for bad in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 7] = bad
        x, xp = both(t, kv, cu)
        assert x[1].isnan().all() and torch.equal(x[::2], o[::2])
        assert xp[40:60].isnan().all() and torch.equal(xp[:40], op[:40]) and torch.equal(xp[60:], op[60:])
    width = table.shape[1] * page
    t = table.clamp_min(0)
    x, xp = both(t, _ints([200, 10 ** 9, -5]), cu)
    y, yp = both(t, _ints([200, width, 0]), cu)
    assert torch.equal(x, y) and torch.equal(xp, yp) and (x[2] == 0).all() and (xp[60:] == 0).all()
    x, xp = both(table, kv, _ints([0, 40, 60, 10 ** 6]))
    assert torch.equal(xp, op)
    x, xp = both(table, kv, _ints([-3, 40, 40, 40]))
    assert torch.equal(xp[:40], op[:40]) and (xp[40:] == 7).all()
    # bounds that fall count as the highest before them
    x, xp = both(table, kv, _ints([0, 40, 20, 90]))
    y, yp = both(table, kv, _ints([0, 40, 40, 90]))
    assert torch.equal(xp, yp)


def test_bounds_that_fall_leave_the_workspace_as_it_was():
    """Many sequences that would all have every row: one has them, and the next calls are right."""
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(3)
    n, B = 700, 80
    q, k, v = (torch.randn((n, h, HD), generator=g, device="cuda").to(BF) for h in (HQ, HKV, HKV))
    want, out = torch.empty_like(q), torch.empty_like(q)
    A.attn_prompt(q, k, v, _ints([0, n]), want)
    bad = _ints([0, n] * (B // 2) + [0])
    A.attn_prompt(q, k, v, bad, out, cu_k=bad)
    torch.cuda.synchronize()
    ref, tol = R.attend(q, k, v, HD ** -0.5, R.causal(n, n, "cuda"), BF)
    R.check(out, ref, tol)
    A.attn_prompt(q, k, v, _ints([0, n]), out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_strided_queries_and_outputs():
    """Queries as columns of the projection, outputs as columns of a wider buffer, and a table that is
    a view; what lies between is left alone."""
    from qwen35_amd.kernels import attention as A
    g = torch.Generator(device="cuda").manual_seed(12)
    T = 70
    proj = torch.randn((T, 2 * HQ * HD + 2 * HKV * HD), generator=g, device="cuda").to(BF)
    q = proj[:, :2 * HQ * HD].view(T, HQ, 2 * HD)[..., :HD]
    wide = torch.full((T, HQ, HD + 64), 7.0, dtype=BF, device="cuda")
    out = wide[..., :HD]
    k0 = 2 * HQ * HD
    k, v = proj[:, k0:k0 + HKV * HD].view(T, HKV, HD), proj[:, k0 + HKV * HD:].view(T, HKV, HD)
    A.attn_prompt(q, k, v, _ints([0, T]), out)
    ref, tol = R.attend(q, k, v, HD ** -0.5, R.causal(T, T, "cuda"), BF)
    R.check(out, ref, tol)
    assert (wide[..., HD:] == 7).all()
    t, pages = R.pages_of([100, 40], 32, 1, 4, "cuda")
    c = R.cache(pages, 32, HKV, HD, BF, 2)
    big = torch.full((4, 50), -1, dtype=torch.int32, device="cuda")
    big[::2, 3:3 + t.shape[1]] = t
    view = big[::2, 3:3 + t.shape[1]]
    out = wide[:2, :, :HD]
    A.attn_decode(q[:2], c[0], c[1], view, _ints([100, 40]), out)
    for b, n in enumerate((100, 40)):
        kk, vv = R.gathered(c, t, b, n)
        ref, tol = R.attend(q[b:b + 1], kk, vv, HD ** -0.5, R.causal(1, n, "cuda"), BF)
        R.check(out[b:b + 1], ref, tol)
    assert (wide[..., HD:] == 7).all()


def test_a_capture_without_a_workspace_is_refused():
    from qwen35_amd.kernels import attention as A
    c = R.cache(4, 16, HKV, HD, BF, 2)
    q = torch.zeros((1, HQ, HD), dtype=BF, device="cuda")
    out, table, n = torch.empty_like(q), _ints([[0, 1]]), _ints([5])
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="without a workspace"):
        with torch.cuda.graph(graph, stream=s):
            A.attn_decode(q, c[0], c[1], table, n, out)
    torch.cuda.synchronize()
