"""A decode step of several candidates of one prompt as the engine would take it: projections, per-head norm with
rotary positions into the cache, attention over the shared prompt, output projection, vocabulary head, penalties
and a grammar's mask, the draw; eager, captured and replayed."""
from __future__ import annotations

import candidates_ref as S
import helpers as H
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HQ, HKV, HD, HID, V, PAGE, PROMPT, B = 8, 2, 256, 1024, 5008, 64, 333, 6


class Step:
    """One attention layer and the vocabulary head over a prompt of PROMPT tokens; the step's inputs and outputs are
    tensors that stay, so that it can be captured."""

    def __init__(self, int8):
        from qwen35_amd.kernels import attention as A
        g = torch.Generator(device="cuda").manual_seed(3)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF)
        w8 = lambda K, N, seed: tuple(t.cuda() for t in H.engine_w8(K, N, seed=seed))
        NQ = 2 * HQ * HD
        self.wq, self.wk, self.wv = w8(HID, NQ, 1), w8(HID, HKV * HD, 2), w8(HID, HKV * HD, 3)
        self.wo, self.head = w8(HQ * HD, HID, 4), w8(HID, V, 5)
        self.in_norm, self.post_norm, self.qn, self.kn = rand(HID) * 0.1, rand(HID) * 0.1, rand(HD) * 0.1, rand(HD) * 0.1
        self.freqs = 1e6 ** -(torch.arange(0, 64, 2, device="cuda", dtype=torch.float64) / 64)
        pages = 6 + 2 * B
        shape = (pages, HKV, PAGE, HD)
        if int8:
            self.kc, self.vc = (torch.zeros(shape, dtype=torch.int8, device="cuda").transpose(1, 2) for _ in range(2))
            self.ks, self.vs = (torch.ones(shape[:3], device="cuda").transpose(1, 2) for _ in range(2))
        else:
            self.kc, self.vc = (torch.zeros(shape, dtype=BF, device="cuda").transpose(1, 2) for _ in range(2))
            self.ks = self.vs = None
        ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.ptable, self.plen, self.cu = torch.arange(6, dtype=torch.int32, device="cuda")[None], ints(PROMPT), ints(0, B)
        self.table = (6 + torch.arange(2 * B, dtype=torch.int32, device="cuda")).view(B, 2).contiguous()
        # the prompt's keys and values, once for all candidates
        k, v = rand(PROMPT, HKV, HD), rand(PROMPT, HKV, HD)
        A.qk_norm_rope(rand(PROMPT, HQ, HD), k, torch.arange(PROMPT, device="cuda"), self.freqs, rand(PROMPT, HQ, HD), v=v,
                       k_cache=self.kc, v_cache=self.vc, slots=torch.arange(PROMPT, device="cuda"), k_s=self.ks, v_s=self.vs,
                       q_w=self.qn, k_w=self.kn)
        # the step's state
        self.hidden, self.u = rand(B, HID), torch.zeros(B, device="cuda")
        self.start = self.hidden.clone()
        self.kv_len, self.slots, self.pos = ints(*[1] * B), torch.zeros(B, dtype=torch.int64, device="cuda"), ints(*[PROMPT] * B)
        self.history = torch.full((B, 64), -1, dtype=torch.int32, device="cuda")
        self.lens, self.plens = ints(*[20] * B), ints(*[15] * B)
        self.history[:, :20] = torch.randint(0, V, (B, 20), generator=g, device="cuda").int()
        self.allowed = torch.rand((B, V), generator=g, device="cuda") < 0.5
        self.bits = S.bits_of(self.allowed)
        empty = lambda *s, dt=BF: torch.empty(s, dtype=dt, device="cuda")
        self.xq, self.xs = empty(B, HID, dt=torch.int8), empty(B, HID // 64, dt=torch.float32)
        self.aq, self.as_ = empty(B, HQ * HD, dt=torch.int8), empty(B, HQ * HD // 64, dt=torch.float32)
        self.proj, self.q, self.out = empty(B, NQ + 2 * HKV * HD), empty(B, HQ, HD), empty(B, HQ, HD)
        self.logits, self.scores = empty(B, V), empty(B, V, dt=torch.float32)
        self.tokens, self.logp = empty(B, dt=torch.int64), empty(B, dt=torch.float32)

    def set(self, n):
        """Before step n (0, 1, ...): positions, places, lengths and uniform numbers."""
        self.kv_len.fill_(n + 1)
        self.pos.fill_(PROMPT + n)
        self.slots.copy_((6 + 2 * torch.arange(B, device="cuda") + n // PAGE) * PAGE + n % PAGE)
        self.lens.fill_(20 + n)
        self.u.copy_(torch.rand(B, generator=torch.Generator().manual_seed(n)))
        self.hidden.copy_(self.start)
        self.hidden[:, 0] += n

    def run(self):
        from qwen35_amd.kernels import attention as A
        from qwen35_amd.kernels import gemm, norm, sampling
        norm.rmsnorm_quant(self.hidden, self.in_norm, self.xq, self.xs)
        gemm.proj3(self.xq, self.xs, *self.wq, *self.wk, *self.wv, self.proj)
        NQ = 2 * HQ * HD
        k = self.proj[:, NQ:NQ + HKV * HD].view(B, HKV, HD)
        v = self.proj[:, NQ + HKV * HD:].view(B, HKV, HD)
        A.qk_norm_rope(self.proj[:, :NQ].view(B, HQ, 2 * HD)[..., :HD], k, self.pos, self.freqs, self.q, v=v, k_cache=self.kc,
                       v_cache=self.vc, slots=self.slots, k_s=self.ks, v_s=self.vs, q_w=self.qn, k_w=self.kn)
        A.attn_decode_shared(self.q, self.kc, self.vc, self.ptable, self.plen, self.cu, self.table, self.kv_len, self.out,
                             k_s=self.ks, v_s=self.vs)
        norm.gate_mul_quant(self.out.view(B, HQ * HD), self.proj[:, :NQ], self.aq, self.as_, hd=HD)
        gemm.gemm_i8(self.aq, self.as_, *self.wo, self.hidden, residual=self.hidden)
        norm.rmsnorm_quant(self.hidden, self.post_norm, self.xq, self.xs)
        gemm.gemm_i8(self.xq, self.xs, *self.head, self.logits)
        sampling.logits_process(self.logits, self.scores, tokens=self.history, lens=self.lens, prompt_lens=self.plens,
                                repetition=1.3, presence=0.5, frequency=0.25, mask=self.bits)
        sampling.sample(self.scores, self.u, self.tokens, logprobs=self.logp, temperature=0.7, top_k=20, top_p=0.9)

    def check(self, n):
        """Every new operator against the formula on the inputs it had."""
        c = S.Batch.__new__(S.Batch)
        c.groups, c.own, c.hkv, c.dt, c.scale = [(B, PROMPT)], [n + 1] * B, HKV, BF, HD ** -0.5
        c.ptable, c.table, c.cache, c.q = self.ptable, self.table, (self.kc, self.vc, self.ks, self.vs), self.q
        c.check(self.out)
        ref, tol = S.logits_formula(self.logits.cpu(), self.history.cpu(), self.lens.cpu(), self.plens.cpu(), 1.3, 0.5, 0.25,
                                    allowed=self.allowed, to=torch.float32)
        y = self.scores.cpu()
        assert torch.equal(y == -torch.inf, ref == -torch.inf)
        # (1.3 is a 32-bit number on the way)
        far = (y.double() - ref).abs().nan_to_num(0, 0, 0) - tol - ref.abs().nan_to_num(0, 0, 0) * 2 ** -23
        assert float(far.max()) <= 0
        f = lambda x: float(torch.tensor(x))
        for b in range(B):
            tok, log, near = S.draw(y[b], float(self.u[b]), 20, f(0.7), f(0.9))
            assert near > 1e-12 and int(self.tokens[b]) == tok
            assert abs(float(self.logp[b]) - log) <= (140 + abs(log)) * S.E32 * 1.01

    def keep(self, n):
        """The drawn tokens, as the next step's history."""
        self.history[:, 20 + n] = self.tokens.int()


@pytest.mark.parametrize("int8", [False, True])
def test_steps(int8):
    from qwen35_amd.kernels import qlin as C
    s = Step(int8)
    s.set(0)
    s.run()
    torch.cuda.synchronize()
    s.check(0)
    graph = torch.cuda.CUDAGraph()
    with C.capture(graph):
        s.run()
    names = ("out", "logits", "scores", "tokens", "logp")
    for n in range(4):
        s.set(n)
        s.run()
        eager = [getattr(s, x).clone() for x in names]
        for x in names:
            getattr(s, x).zero_()
        s.set(n)
        graph.replay()
        torch.cuda.synchronize()
        for x, e in zip(names, eager):
            assert torch.equal(getattr(s, x), e), (n, x)
        s.check(n)
        assert bool(s.allowed.gather(1, s.tokens[:, None]).all())
        s.keep(n)
