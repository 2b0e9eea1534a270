"""logits_process with more biases or longer histories than a word for each token holds (4094 of a row, 2^19 - 1 tokens), and
with as many as it does."""
from __future__ import annotations

import math

import candidates_ref as S
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(x, to, **kw):
    from qwen35_amd.kernels import sampling
    on = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    return sampling.logits_process(x.cuda(), torch.full(x.shape, 9.0, dtype=to, device="cuda"), **on).cpu()


def check(y, ref, tol):
    hidden = ref == -math.inf
    assert torch.equal(y == -math.inf, hidden)
    bad = ~((y.double() - ref).abs() <= tol) & ~hidden
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())


def biases(B, V, nb, seed):
    """Ids that repeat, in every distance from each other, and ids outside the vocabulary."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (B, nb), generator=g)
    ids[:, ::5] = ids[:, :1]                                  # one id all along
    few = min(40, nb // 2)
    ids[:, nb // 2:nb // 2 + few] = torch.arange(few) // 2    # neighbours twice
    ids[:, 7::211] = -1
    ids[:, 9::211] = V
    ids[:, -1] = V - 1                                        # the last place of all, in a row's tail
    ids[0, 0] = V - 1
    return ids.int(), torch.randn((B, nb), generator=g) * 5


@pytest.mark.parametrize("nb", [4094, 4095, 5000])
@pytest.mark.parametrize("V", [41, 4099, 20011])
@pytest.mark.parametrize("history", [0, 300])
@pytest.mark.parametrize("dt,to", [(BF, F32), (F32, F16)])
def test_many_biases(nb, V, history, dt, to):
    B = 3
    g = torch.Generator().manual_seed(nb + V)
    x = (torch.randn((B, V), generator=g) * 4).to(dt)
    ids, bias = biases(B, V, nb, nb)
    allowed = torch.rand((B, V), generator=g) < 0.8
    kw, ref = {}, {}
    if history:
        t = torch.randint(-1, V + 1, (B, history), generator=g)
        t[:, ::3] = ids[:, 1:2].long()                         # a token of the history with a bias
        p, r = torch.tensor([0, 100, 300]).int(), 1 + torch.rand(B, generator=g)
        kw = dict(tokens=t, prompt_lens=p, repetition=r, presence=0.5, frequency=0.25)
        ref = dict(tokens=t, prompt=p, rep=r, pres=0.5, freq=0.25)
    ref, tol = S.logits_formula(x, ids=ids, bias=bias, allowed=allowed, to=to, **ref)
    for mask in (S.bits_of(allowed), allowed):
        check(run(x, to, bias_ids=ids, bias=bias, mask=mask, **kw), ref, tol)


@pytest.mark.parametrize("L", [(1 << 19) - 1, 1 << 19, (1 << 19) + 77])
@pytest.mark.parametrize("nb", [0, 17, 4500])
def test_a_long_history_with_biases(L, nb):
    """One token as often as a word can count, others a few times, with the place of a bias beside the count."""
    V, B = 3000, 2
    g = torch.Generator().manual_seed(L + nb)
    x = torch.randn((B, V), generator=g) * 4
    t = torch.full((B, L), 17, dtype=torch.int32)
    t[1, 5::1000] = torch.randint(0, V, (len(range(5, L, 1000)),), generator=g).int()
    prompt = torch.tensor([0, L // 2]).int()
    kw, ref = {}, {}
    if nb:
        ids, bias = biases(B, V, nb, L)
        ids[:, nb // 2] = 17
        kw, ref = dict(bias_ids=ids, bias=bias), dict(ids=ids, bias=bias)
    ref, tol = S.logits_formula(x, t, None, prompt, 1.25, 0.5, 2.0 ** -10, to=F32, **ref)
    check(run(x, F32, tokens=t, prompt_lens=prompt, repetition=1.25, presence=0.5, frequency=2.0 ** -10, **kw), ref, tol)


@pytest.mark.parametrize("nb", [4094, 4095])
def test_the_last_of_one_id(nb):
    """All of a row's biases are one id's, or two ids' in turn."""
    x = torch.zeros((2, 100))
    ids = torch.full((2, nb), 31, dtype=torch.int32)
    ids[1, ::2] = 99
    bias = torch.arange(nb).float().expand(2, -1).contiguous()
    y = run(x, F32, bias_ids=ids, bias=bias)
    want = torch.zeros((2, 100))
    want[0, 31] = nb - 1
    last = [i for i in range(nb) if i % 2 == 0][-1]
    want[1, 99], want[1, 31] = last, nb - 1 if last != nb - 1 else nb - 2
    assert torch.equal(y, want)
