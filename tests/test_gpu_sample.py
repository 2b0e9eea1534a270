"""sample against the formula in 64 bits (candidates_ref.py).

Tokens have to be equal: the kernel's weights and sums are of 64 bits, so that only a draw within 1e-12 of
a border could fall otherwise (none of these does; the tests look).  Log probabilities: the row's sum of n
exponentials in 32 bits, each with an error of (|x - max| log2(e) + 2) e (the argument's rounding, and
the exponential's) relative to itself, which with at most 96 steps a number is added through gives a relative
error below (96 + 4 + 40) e of the sum (larger arguments than 40 weigh nothing), hence of its logarithm
absolutely; and half a step of the result."""
from __future__ import annotations

import math

import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(x, u, tok=torch.int64, logprobs=True, **kw):
    from qwen35_amd.kernels import sampling
    tokens = torch.full((x.shape[0],), 99, dtype=tok, device="cuda")
    lp = torch.full((x.shape[0],), 99.0, device="cuda") if logprobs else None
    assert sampling.sample(x, u, tokens, logprobs=lp, **kw) is tokens
    return tokens.cpu(), None if lp is None else lp.cpu()


def check(x, u, top_k=20, temperature=1.0, top_p=1.0, min_p=0.0, **kw):
    """x, u on the CPU."""
    on = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v
    tok, lp = run(x.cuda(), u.cuda(), top_k=top_k, temperature=on(temperature), top_p=on(top_p), min_p=on(min_p), **kw)
    row = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else float(torch.tensor(v, dtype=F32))
    for b in range(x.shape[0]):
        want, log, near = S.draw(x[b], float(u[b]), top_k, row(temperature, b), row(top_p, b), row(min_p, b))
        assert near > 1e-12, (b, near)
        assert int(tok[b]) == want, (b, int(tok[b]), want, near)
        if math.isinf(log):
            assert float(lp[b]) == log
        else:
            assert abs(float(lp[b]) - log) <= 140 * S.E32 + abs(log) * S.E32 * 1.01, (b, float(lp[b]), log)
    return tok


def rows(B, V, seed, dt=F32, sd=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((B, V), generator=g) * sd).to(dt), torch.rand(B, generator=g)


@pytest.mark.parametrize("V", [1, 2, 20, 127, 500, 8192, 8193, 50021])
@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_sizes(V, dt, k):
    x, u = rows(4, V, V + k, dt)
    check(x, u, top_k=k, temperature=0.8, top_p=0.9, min_p=0.01)


@pytest.mark.parametrize("V,k", [(248320, 20), (248320, 128), (300000, 128), (700001, 100)])
def test_whole_vocabularies(V, k):
    """Tiles of a row on many workgroups; more tiles than lists can be joined."""
    x, u = rows(2, V, 5, F32)
    check(x, u, top_k=k)
    check(x.to(BF), u, top_k=k, temperature=2.0)          # many of equal value


def test_many_rows():
    x, u = rows(300, 9001, 7, BF)
    g = torch.Generator().manual_seed(8)
    t, p, m = (torch.rand(300, generator=g) for _ in range(3))
    t[::7] = 0.0
    t[3] = -1.0                                            # counts as 0
    want = t.clamp_min(0)
    tok, _ = run(x.cuda(), u.cuda(), temperature=t.cuda(), top_p=p.cuda(), min_p=m.cuda() * 0.2, top_k=40)
    got = check(x, u, temperature=want, top_p=p, min_p=m * 0.2, top_k=40)
    assert torch.equal(tok, got)


def test_values_in_every_order():
    """Rows whose largest lie together, in one thread's places, in the last tile, ascending, descending, all equal."""
    V = 8192 * 3 + 5
    i = torch.arange(V)
    x = torch.stack([i.float(), -i.float(), torch.zeros(V), (i % 2048 < 8).float() * 50 + i * 1e-4,
                     (i % 8192 % 2048 // 8 < 128).float() * 90 + (i % 97), torch.where(i > 2 * 8192, i, 0).float(),
                     (i == 8192).float() * 30, -(i % 251).float()]) * 0.25
    for k in (1, 64, 128):
        for at in (0.0, 0.4, 0.999):
            check(x, torch.full((8,), at + 1e-4), top_k=k, temperature=3.0)


@pytest.mark.parametrize("dt", [BF, F32])
def test_ties_go_to_the_lowest_index(dt):
    x = torch.full((1, 30000), 1.5, dtype=dt)
    x[0, 20000] = 2.0
    for n, want in ((1, 20000), (2, 0), (3, 1), (100, 98)):
        tok, _ = run(x.cuda(), torch.tensor([1 - 2.0 ** -24]).cuda(), top_k=n)
        assert int(tok) == want
    x[0, 5] = -0.0
    x[0, :5] = -1
    x[0, 6:] = -2
    x[0, 9] = 0.0                                          # equal to -0
    tok, _ = run(x.cuda(), torch.tensor([0.0]).cuda(), top_k=2)
    assert int(tok) == 5


def test_frequencies():
    """Evenly spread draws meet each token as often as its probability says."""
    V, n = 1000, 4096
    g = torch.Generator().manual_seed(3)
    x = torch.randn(V, generator=g) * 2
    u = (torch.arange(n) + 0.5) / n
    tok, _ = run(x.cuda().expand(n, V), u.cuda(), top_k=50, top_p=0.9, temperature=1.3)
    val, ids = torch.sort(x.double(), descending=True)
    p = torch.softmax(val[:50] / float(torch.tensor(1.3)), 0)
    kept = int((p.cumsum(0) - p < float(torch.tensor(0.9))).sum())
    p = p[:kept] / p[:kept].sum()
    got = torch.bincount(tok, minlength=V)[ids].double() / n
    assert float(got[kept:].sum()) == 0
    assert float((got[:kept] - p).abs().max()) <= 1.01 / n


def test_masked_rows():
    """Rows that leave fewer tokens than top_k, one, or none; NaN is never drawn."""
    x, _ = rows(6, 20000, 9)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 12345] = -4.0
    x[2, 3:] = -math.inf
    x[3] = math.nan
    x[4, ::2] = math.nan
    x[5] = torch.finfo(F32).min                            # the type's lowest value is a value
    for at in (0.0, 0.5, 0.999):
        tok = check(torch.where(x.isnan(), -math.inf, x), torch.full((6,), at) + 1e-3 * (at == 0.5), temperature=0.7)
        same, _ = run(x.cuda(), (torch.full((6,), at) + 1e-3 * (at == 0.5)).cuda(), temperature=0.7)
        assert torch.equal(tok, same)
        assert tok[0] == -1 and tok[1] == 12345 and tok[3] == -1


def test_infinite_logits_share_the_row():
    x, _ = rows(2, 9000, 10)
    x[0, [70, 8500]] = math.inf
    x[1, 4] = math.inf
    for at, want in ((0.0, 70), (0.49, 70), (0.51, 8500), (0.99, 8500)):
        for t in (0.0, 0.7):
            tok, lp = run(x.cuda(), torch.tensor([at, at]).cuda(), temperature=t)
            assert tok.tolist() == [want, 4]
            assert abs(float(lp[0]) + math.log(2)) < 1e-6 and float(lp[1]) == 0


def test_uniform_numbers_outside_their_range():
    x = torch.tensor([[0.0, 3.0, 2.0, 1.0]] * 4, device="cuda")
    tok, _ = run(x, torch.tensor([-1.0, 1.0, 7.0, math.nan]).cuda(), top_k=3)
    assert tok.tolist() == [1, 3, 3, 3]


def test_options():
    x, u = rows(3, 777, 11, F16)
    tok, lp = run(x.cuda(), u.cuda(), tok=torch.int32)
    same, none = run(x.cuda(), u.cuda(), logprobs=False)
    assert none is None and torch.equal(tok.long(), same)
    room = torch.zeros((3, 1000), dtype=F16)
    room[:, 13:790] = x                                    # rows at odd addresses
    again, lp2 = run(room.cuda()[:, 13:790], u.cuda())
    assert torch.equal(again, same) and torch.equal(lp, lp2)
    greedy, _ = run(x.cuda(), u.cuda(), temperature=0.0)
    assert torch.equal(greedy, x.float().argmax(1))
    first, _ = run(x.cuda(), u.cuda(), top_p=0.0)
    assert torch.equal(first, greedy)
    first, _ = run(x.cuda(), u.cuda(), min_p=1.0)
    assert torch.equal(first, greedy)


def test_empty_batch():
    run(torch.empty((0, 5), device="cuda"), torch.empty(0, device="cuda"))


def test_graph_and_streams():
    from qwen35_amd.kernels import qlin as C
    from qwen35_amd.kernels import sampling
    x, u = rows(9, 60000, 12)
    xc, uc = x.cuda(), u.cuda()
    tokens, lp = torch.empty(9, dtype=torch.int64, device="cuda"), torch.empty(9, device="cuda")
    sampling.sample(xc, uc, tokens, logprobs=lp)
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        sampling.sample(xc, uc, tokens, logprobs=lp)
    for i in range(4):
        y, v = rows(9, 60000, 13 + i)
        xc.copy_(y), uc.copy_(v)
        eager = run(xc, uc)
        tokens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens.cpu(), eager[0]) and torch.equal(lp.cpu(), eager[1])
        assert torch.equal(check(y, v), eager[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        C.bind_workspace(s)
    outs = []
    torch.cuda.synchronize()
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                t = torch.empty(9, dtype=torch.int64, device="cuda")
                outs.append(sampling.sample(xc, uc, t))
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), eager[0]) for o in outs)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_many_of_equal_value(dt, k):
    """Masks of the type's lowest value, rows of a few distinct values, and ties at the k-th place."""
    V = 8192 * 4 + 77
    g = torch.Generator().manual_seed(k)
    low = torch.finfo(dt).min
    x = torch.full((5, V), low, dtype=dt)
    x[0, torch.randperm(V, generator=g)[:k // 2 + 1]] = 1.0           # the others come from the masked ones
    x[1] = torch.randint(0, 3, (V,), generator=g).to(dt)
    x[2] = torch.randint(0, 300, (V,), generator=g).to(dt)
    x[3, 9000:] = -2.5
    x[4] = (torch.arange(V) % 8 == 5).to(dt)                          # one place of each thread's eight
    for u in (0.1, 0.9):
        check(x, torch.full((5,), u), top_k=k, temperature=1e9 if dt == F32 else 2.0)


def test_most_in_few_threads():
    """A tile whose largest lie in 100 threads' places, all different: more than reach the list as a rule."""
    V = 8192 + 100
    i = torch.arange(V)
    x = torch.where(i % 2048 < 800, 50 + (i * 2654435761 % 4096).float() / 128, -i.float() / 4096)[None].expand(3, V).contiguous()
    x[1, 8192:] = 200.0
    for k in (50, 128):
        for u in (0.001, 0.77, 0.9999):
            check(x, torch.full((3,), u), top_k=k, temperature=20.0)


@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("B,V,k", [(16, 262145, 128), (24, 248320, 40), (40, 131073, 5), (20, 300001, 100)])
def test_long_parts(B, V, k, dt):
    """Many rows of long vocabularies: parts of up to 16384 logits, or longer ones that are read twice."""
    x, u = rows(B, V, B + k, dt)
    check(x, u, top_k=k, temperature=0.9, top_p=0.95)
