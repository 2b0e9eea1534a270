"""logits_process against the formula in 64 bits (candidates_ref.py)."""
from __future__ import annotations

import math

import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def P(*a, **kw):
    from qwen35_amd.kernels import sampling
    return sampling.logits_process(*a, **kw)


def _rows(B, V, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, V), generator=g) * 4).to(dt)


def _history(B, V, L, seed, dt=torch.int32):
    """Histories that repeat few tokens often, of all lengths, with padding of both kinds."""
    g = torch.Generator().manual_seed(seed)
    t = (torch.rand((B, L), generator=g) ** 4 * V).long()
    t[:, ::7] = t[:, :1]
    pad = torch.rand((B, L), generator=g)
    t[pad < 0.05] = -1
    t[pad > 0.95] = V
    lens = torch.randint(0, L + 1, (B,), generator=g)
    lens[0] = L
    prompt = (lens * torch.rand(B, generator=g)).long()
    return t.to(dt), lens.int(), prompt.int()


def _check(y, ref, tol, to):
    y = y.cpu()
    assert y.dtype == to
    inf = ref == -math.inf
    assert torch.equal(y == -math.inf, inf)
    err = (y.double() - ref).abs()
    bad = ~(err <= tol) & ~inf
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), float(err[bad].max()))


@pytest.mark.parametrize("V", [1, 7, 8, 33, 2047, 2048, 2049, 8192, 8195, 50021])
@pytest.mark.parametrize("dt,to", [(BF, F32), (F16, F16), (F32, F32), (F32, BF), (BF, F16)])
def test_all_at_once(V, dt, to):
    B, L, nb = 3, 200, 9
    x = _rows(B, V, dt, V)
    t, lens, prompt = _history(B, V, L, V + 1)
    g = torch.Generator().manual_seed(V + 2)
    rep, pres, freq = 1 + torch.rand(B, generator=g), torch.rand(B, generator=g) * 2, torch.randn(B, generator=g)
    ids = torch.randint(-2, V + 2, (B, nb), generator=g).int()
    bias = torch.randn((B, nb), generator=g) * 5
    allowed = torch.rand((B, V), generator=g) < 0.7
    ref, tol = S.logits_formula(x, t, lens, prompt, rep, pres, freq, ids, bias, allowed, to)
    cu = lambda *ts: [a.cuda() for a in ts]
    xc, tc, lc, pc, rc, sc, fc, ic, bc, ac = cu(x, t, lens, prompt, rep, pres, freq, ids, bias, allowed)
    for mask in (S.bits_of(allowed).cuda(), ac):
        out = torch.full((B, V), 9.0, dtype=to, device="cuda")
        y = P(xc, out, tokens=tc, lens=lc, prompt_lens=pc, repetition=rc, presence=sc, frequency=fc, bias_ids=ic,
              bias=bc, mask=mask)
        assert y is out
        _check(y, ref, tol, to)


@pytest.mark.parametrize("which", ["nothing", "repetition", "presence", "frequency", "prompt", "bias", "mask"])
def test_one_at_a_time(which):
    B, V, L = 4, 5003, 60
    x = _rows(B, V, BF, 3)
    t, lens, prompt = _history(B, V, L, 4, torch.int64)
    g = torch.Generator().manual_seed(5)
    ref_kw, kw = {}, {}
    if which in ("repetition", "presence", "frequency"):
        kw = {which: 1.3, "tokens": t.cuda()}
        ref_kw = {{"repetition": "rep", "presence": "pres", "frequency": "freq"}[which]: 1.3, "tokens": t}
    elif which == "prompt":
        kw = dict(tokens=t.cuda(), prompt_lens=prompt.cuda(), presence=-0.7, repetition=0.8)
        ref_kw = dict(tokens=t, prompt=prompt, pres=-0.7, rep=0.8)
    elif which == "bias":
        ids = torch.randint(0, V, (B, 700), generator=g).int()
        bias = torch.randn((B, 700), generator=g)
        kw, ref_kw = dict(bias_ids=ids.cuda(), bias=bias.cuda()), dict(ids=ids, bias=bias)
    elif which == "mask":
        allowed = torch.rand((1, V), generator=g) < 0.01          # one mask for all rows
        kw, ref_kw = dict(mask=S.bits_of(allowed).cuda().expand(B, -1)), dict(allowed=allowed.expand(B, -1))
    ref, tol = S.logits_formula(x, **ref_kw, to=F32)
    # (numbers that are given as one for all are 32-bit ones on the way)
    tol = tol + ref.abs().nan_to_num(0, 0, 0) * 2 ** -22
    _check(P(x.cuda(), torch.empty((B, V), device="cuda"), **kw), ref, tol, F32)
    if which == "nothing":
        assert torch.equal(P(x.cuda(), torch.empty((B, V), device="cuda")).cpu(), x.float())
        y = x.cuda()
        assert torch.equal(P(y, y).cpu(), x)


@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("V", [5, 4099])
def test_in_place_is_the_same(dt, V):
    x = _rows(5, V, dt, 7).cuda()
    t, lens, prompt = (a.cuda() for a in _history(5, V, 99, 8))
    kw = dict(tokens=t, lens=lens, prompt_lens=prompt, repetition=1.2, presence=0.5, frequency=0.25)
    want = P(x, torch.empty_like(x), **kw)
    room = torch.full((5, V + 11), 3.0, dtype=dt, device="cuda")
    room[:, 2:2 + V] = x
    P(room[:, 2:2 + V], room[:, 2:2 + V], **kw)
    assert torch.equal(room[:, 2:2 + V], want)
    assert bool((room[:, :2] == 3).all()) and bool((room[:, 2 + V:] == 3).all())


def test_rows_between_rows():
    """Inputs and outputs whose rows lie between each other's, at odd addresses."""
    V, B = 1001, 4
    x = _rows(B, V, BF, 9)
    both = torch.full((B, 2 * V + 1), 5.0, dtype=BF, device="cuda")
    both[:, 1 + V:] = x.cuda()
    ref, tol = S.logits_formula(x, allowed=(x > 0), to=BF)
    P(both[:, 1 + V:], both[:, 1:1 + V], mask=S.bits_of(x > 0).cuda())
    _check(both[:, 1:1 + V], ref, tol, BF)
    assert bool((both[:, 0] == 5).all()) and torch.equal(both[:, 1 + V:].cpu(), x)


def test_a_long_history_of_one_token():
    """Counts are exact whole numbers up to the 24 bits that 32-bit numbers hold."""
    V, L = 300, 1 << 20
    t = torch.full((2, L), 17, dtype=torch.int32)
    t[1, 5::2] = 40
    x = torch.ones((2, V))
    y = P(x.cuda(), torch.empty((2, V), device="cuda"), tokens=t.cuda(), prompt_lens=torch.tensor([3, 0]).int().cuda(),
          frequency=0.5, lens=torch.tensor([L, L]).int().cuda()).cpu()
    n40 = len(range(5, L, 2))
    assert y[0, 17] == 1 - 0.5 * (L - 3) and y[1, 40] == 1 - 0.5 * n40 and y[1, 17] == 1 - 0.5 * (L - n40)
    assert int((y != 1).sum()) == 3


def test_lengths_outside_the_history():
    V = 50
    t = torch.arange(10, dtype=torch.int32).expand(4, 10).contiguous().cuda()
    x = torch.ones((4, V), device="cuda")
    lens = torch.tensor([-5, 0, 1 << 30, 3], dtype=torch.int32, device="cuda")
    prompt = torch.tensor([0, 4, -3, 1 << 30], dtype=torch.int32, device="cuda")
    y = P(x, torch.empty_like(x), tokens=t, lens=lens, prompt_lens=prompt, presence=2.0, repetition=4.0)
    want = torch.ones((4, V))
    want[2, :10] = 0.25 - 2
    want[3, :3] = 0.25
    assert torch.equal(y.cpu(), want)


def test_biases():
    """Of an id that is given twice the last counts; infinite biases ban and force; the mask comes last."""
    V = 100
    ids = torch.tensor([[3, 5, 3, -1, 100, 7, 8, 9, 3]], dtype=torch.int32, device="cuda")
    b = torch.tensor([[1.0, 2, 4, 99, 99, -math.inf, math.inf, math.inf, 8]], device="cuda")
    x = torch.ones((1, V), device="cuda")
    allowed = torch.ones((1, V), dtype=torch.bool, device="cuda")
    allowed[0, 9] = False
    y = P(x, torch.empty_like(x), bias_ids=ids, bias=b, mask=allowed).cpu()[0]
    assert y[3] == 9 and y[5] == 3 and y[7] == -math.inf and y[8] == math.inf and y[9] == -math.inf
    assert int((y != 1).sum()) == 5


def test_odd_values():
    """Infinities and NaN go through the formulas; where the mask hides them they are gone."""
    V = 64
    x = torch.ones((1, V), device="cuda")
    x[0, :6] = torch.tensor([math.nan, math.inf, -math.inf, math.nan, math.inf, torch.finfo(F32).min])
    t = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    allowed = torch.ones((1, V), dtype=torch.bool, device="cuda")
    allowed[0, 3:5] = False
    y = P(x, torch.empty_like(x), tokens=t, repetition=2.0, presence=1.0, mask=S.bits_of(allowed)).cpu()[0]
    assert y[0].isnan() and y[1] == math.inf and (y[2:6] == -math.inf).all() and (y[6:] == 1).all()


def test_empty():
    x = torch.empty((0, 10), device="cuda")
    P(x, torch.empty_like(x))
    x = torch.ones((2, 0), device="cuda")
    P(x, torch.empty_like(x))
    x = torch.ones((2, 5), device="cuda")
    none = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    y = P(x, torch.empty_like(x), tokens=none, repetition=3.0, bias_ids=none, bias=none.float())
    assert torch.equal(y, x)


def test_many_rows_and_graph():
    from qwen35_amd.kernels import qlin as C
    B, V, L = 70, 20011, 300
    x = _rows(B, V, BF, 11)
    t, lens, prompt = _history(B, V, L, 12)
    g = torch.Generator().manual_seed(13)
    rep = 1 + torch.rand(B, generator=g)
    xc, tc, lc, pc, rc = (a.cuda() for a in (x, t, lens, prompt, rep))
    out = torch.empty((B, V), device="cuda")
    kw = dict(tokens=tc, lens=lc, prompt_lens=pc, repetition=rc, frequency=0.125)
    P(xc, out, **kw)
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        P(xc, out, **kw)
    for n in (L, 10, 0):
        lens = lens.clamp_max(n)
        lc.copy_(lens)
        eager = P(xc, torch.empty_like(out), **kw).clone()
        out.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        _check(out, *S.logits_formula(x, t, lens, prompt, rep, freq=0.125, to=F32), F32)
