"""Calls of a step of several candidates that a program may make besides the plain ones: pages given twice, one row for all,
views between other data, graphs that share a stream's workspace, threads, the largest batches."""
from __future__ import annotations

import threading

import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("n", [3, 20])
@pytest.mark.parametrize("int8", [False, True])
def test_pages_given_twice(n, int8):
    """A page may be many times in a prefix, in several prefixes and among sequences' own."""
    c = S.Batch([(n, 200), (n, 130)], [50] * (2 * n), 8, 2, 128, BF, seed=5, page=16, int8=int8)
    c.ptable[0, 3] = c.ptable[0, 1]
    c.ptable[1, :4] = c.ptable[0, :4]
    c.table[:, 0] = c.ptable[0, 0]
    c.table[1, 2] = c.table[1, 1]
    c.run()
    c.check(c.out)


def test_one_table_row_for_all():
    """An expanded table (stride 0): all sequences see the same own keys, as many as their lengths say."""
    c = S.Batch([(4, 77)], [40, 1, 33, 0], 8, 2, 64, F16, seed=6, page=16)
    c.table = c.table[:1].expand(4, -1)
    c.run()
    c.check(c.out)


def test_two_graphs_of_one_stream():
    """Graphs captured on one stream share its workspace: replayed in turn, with eager calls between, each gives the eager
    call's bits."""
    from qwen35_amd.kernels import qlin as C
    from qwen35_amd.kernels import sampling
    a = S.Batch([(6, 900), (2, 64)], [30 + i for i in range(8)], 8, 2, 256, BF, seed=7)
    b = S.Batch([(40, 500)], [9] * 40, 16, 2, 128, F16, seed=8)
    g = torch.Generator(device="cuda").manual_seed(9)
    x, y = (torch.randn((r, v), generator=g, device="cuda") * 3 for r, v in ((3, 50021), (70, 9001)))
    u, w = torch.rand(3, generator=g, device="cuda"), torch.rand(70, generator=g, device="cuda")
    t, s = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(70, dtype=torch.int32, device="cuda")
    steps = [lambda: (a.run(), sampling.sample(x, u, t, top_k=40)), lambda: (b.run(), sampling.sample(y, w, s, top_k=100))]
    outs = [(a.out, t), (b.out, s)]
    want = []
    for f, o in zip(steps, outs):
        f()
        want.append([v.clone() for v in o])
    graphs = [torch.cuda.CUDAGraph() for _ in steps]
    for graph, f in zip(graphs, steps):
        with C.capture(graph):
            f()
    for turn in (0, 1, 1, 0, 1, 0):
        for o in outs[turn]:
            o.zero_()
        graphs[turn].replay()
        torch.cuda.synchronize()
        for o, v in zip(outs[turn], want[turn]):
            assert torch.equal(o, v)
        steps[1 - turn]()
        torch.cuda.synchronize()
        for o, v in zip(outs[1 - turn], want[1 - turn]):
            assert torch.equal(o, v)


def test_threads_on_their_own_streams():
    from qwen35_amd.kernels import sampling
    work = []
    for i in range(4):
        c = S.Batch([(5, 700 + i)], [20] * 5, 8, 2, 128, BF, seed=20 + i)
        x = torch.randn((5, 20011), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda") * 3
        u, t, o = torch.full((5,), 0.4, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda"), torch.empty_like(x)
        h = torch.randint(0, 20011, (5, 50), device="cuda")
        work.append((c, x, u, t, o, h))

    def step(c, x, u, t, o, h):
        c.run()
        sampling.logits_process(x, o, tokens=h, repetition=1.2, frequency=0.1)
        sampling.sample(o, u, t)

    want = []
    for w in work:
        step(*w)
        want.append([v.clone() for v in (w[0].out, w[4], w[3])])
        for v in (w[0].out, w[4], w[3]):
            v.zero_()
    torch.cuda.synchronize()
    errors = []

    def many(w, v):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    step(*w)
                torch.cuda.current_stream().synchronize()
            for got, x in zip((w[0].out, w[4], w[3]), v):
                assert torch.equal(got, x)
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=many, args=a) for a in zip(work, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("dt", [BF, F32])
def test_one_row_of_logits_for_all(dt):
    from qwen35_amd.kernels import sampling
    row = (torch.randn((1, 5003), generator=torch.Generator().manual_seed(2)) * 3).to(dt)
    x, u = row.cuda().expand(6, -1), torch.tensor([0.0, 0.2, 0.4, 0.6, 0.8, 0.99])
    t = torch.zeros(6, dtype=torch.int64, device="cuda")
    sampling.sample(x, u.cuda(), t, temperature=0.9, top_k=30)
    for b in range(6):
        tok, _, near = S.draw(row[0], float(u[b]), 30, float(torch.tensor(0.9)))
        assert near > 1e-12 and int(t[b]) == tok
    allowed = torch.rand((1, 5003), generator=torch.Generator().manual_seed(3)) < 0.5
    h = torch.arange(600)[None].expand(6, -1)
    out = torch.empty((6, 5003), device="cuda")
    sampling.logits_process(x, out, tokens=h.cuda()[:1].expand(6, -1), repetition=1.5, mask=allowed.cuda().expand(6, -1))
    ref, tol = S.logits_formula(row.expand(6, -1), h, None, None, 1.5, allowed=allowed.expand(6, -1), to=F32)
    y = out.cpu()
    assert torch.equal(y == -torch.inf, ref == -torch.inf)
    assert float(((y.double() - ref).abs().nan_to_num(0, 0, 0) - tol).max()) <= 0


def test_columns_of_a_wider_tensor():
    """Logits, scores, masks and histories that are columns of wider rows; what lies beside stays as it was."""
    from qwen35_amd.kernels import sampling
    g = torch.Generator().manual_seed(4)
    wide = (torch.randn((5, 4099), generator=g) * 3).to(BF)
    hist = torch.randint(-1, 4001, (5, 90), generator=g)
    allowed = torch.rand((5, 4010), generator=g) < 0.7
    out = torch.full((5, 4021), 7.0, device="cuda")
    x, o = wide.cuda()[:, 3:4004], out[:, 5:4006]
    sampling.logits_process(x, o, tokens=hist.cuda()[:, 7:60], presence=0.75, mask=allowed.cuda()[:, 1:4002])
    ref, tol = S.logits_formula(wide[:, 3:4004], hist[:, 7:60], None, None, 1.0, 0.75, 0.0, allowed=allowed[:, 1:4002], to=F32)
    y = o.cpu()
    assert torch.equal(y == -torch.inf, ref == -torch.inf)
    assert float(((y.double() - ref).abs().nan_to_num(0, 0, 0) - tol).max()) <= 0
    assert bool((out[:, :5] == 7.0).all()) and bool((out[:, 4006:] == 7.0).all())
    u, t = torch.rand(5, generator=g), torch.zeros(5, dtype=torch.int32, device="cuda")
    sampling.sample(o, u.cuda(), t, top_k=7)
    for b in range(5):
        tok, _, near = S.draw(y[b], float(u[b]), 7)
        assert near > 1e-12 and int(t[b]) == tok


def test_most_rows():
    """2^16 rows, on one workgroup each and on two; every row's token is one of its k largest, and all draws from rows that
    hold the same numbers with the same uniform number are one."""
    from qwen35_amd.kernels import sampling
    B = 1 << 16
    for V in (300, 8500):
        base = torch.randn((64, V), generator=torch.Generator().manual_seed(V)) * 3
        x = base.to(BF).cuda().repeat(B // 64, 1)
        u = torch.rand(64, generator=torch.Generator().manual_seed(V + 1))
        t, lp = torch.zeros(B, dtype=torch.int64, device="cuda"), torch.zeros(B, device="cuda")
        sampling.sample(x, u.cuda().repeat(B // 64), t, logprobs=lp, top_k=10, temperature=1.1)
        t, lp = t.view(-1, 64).cpu(), lp.view(-1, 64).cpu()
        assert bool((t == t[0]).all()) and bool((lp == lp[0]).all())
        for b in range(64):
            tok, _, near = S.draw(base[b].to(BF), float(u[b]), 10, float(torch.tensor(1.1)))
            assert near > 1e-12 and int(t[0, b]) == tok
        del x
