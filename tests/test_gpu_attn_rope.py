"""qk_norm_rope against its formula in 64 bits.

Allowed: half a step of the output's type, and in 32 bits the norm (hd / 8 products a lane,
their butterfly, a root and three products: under 16 e in all), a cosine and sine each
within 2^-22 (argument rounded at up to pi, 2 ulp), two products and a sum: 32 e of the pair's
magnitudes.  A code is within half a step of the scale of what it stands for, and its scale
within 2^-19 of amax / 127.
"""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _axis(half, sections, inter):
    if inter:
        n = len(sections)
        return [i % n if i < n * sections[i % n] else 0 for i in range(half)]
    return [a for a, s in enumerate(sections) for _ in range(s)]


def _ref(x, w, eps, one_plus, pos, freqs, axis):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (w.double() + 1 if one_plus else w.double())
    half = freqs.shape[0]
    if half == 0:
        return y, y.abs() * 32 * R.E32
    ang = torch.stack([pos[a].double() * freqs[i].double() for i, a in enumerate(axis)], -1)[:, None]
    a, b = y[..., :half], y[..., half:2 * half]
    out = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), y[..., 2 * half:]], -1)
    mag = torch.cat([a.abs() + b.abs()] * 2 + [y[..., 2 * half:].abs()], -1)
    return out, mag * 32 * R.E32


def _inputs(T, hq, hkv, hd, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    proj = torch.randn((T, 2 * hq * hd + 2 * hkv * hd), generator=g, device="cuda").to(dt)
    q = proj[:, :2 * hq * hd].view(T, hq, 2 * hd)[..., :hd]
    k = proj[:, 2 * hq * hd:(2 * hq + hkv) * hd].view(T, hkv, hd)
    v = proj[:, (2 * hq + hkv) * hd:].view(T, hkv, hd)
    return q, k, v, g


@pytest.mark.parametrize("T", [1, 3, 130])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 32), (256, 64), (256, 256)])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("axes,inter", [(1, False), (2, False), (3, False), (3, True)])
def test_against_the_formula(T, hd, rot, dt, int8, axes, inter):
    from qwen35_amd.kernels import attention as A
    hq, hkv, page = 6, 3, 16
    q, k, v, g = _inputs(T, hq, hkv, hd, dt, T + hd + axes)
    half = rot // 2
    sections = [half - (axes - 1) * (half // 3)] + [half // 3] * (axes - 1)
    pos = torch.randint(0, 250000, (axes, T), generator=g, device="cuda")
    if T % 2:
        pos = pos.int()
    freqs = torch.tensor([1e7 ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
    if rot == 32:
        freqs = freqs.float()
    wq, wk = (torch.randn((hd,), generator=g, device="cuda").to(torch.float32 if rot == 64 else dt) * 0.3
              for _ in range(2))
    pages = T // page + 2
    c = R.cache(pages, page, hkv, hd, dt, 5, int8)
    old = [None if x is None else x.clone() for x in c]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].clone()
    slots[T // 2] = -1 if T > 1 else slots[0]
    if T > 100:
        slots[100] = pages * page        # past the cache
        slots = slots.int()
    q_out = torch.empty((T, hq, hd), dtype=dt, device="cuda")
    k_out = torch.empty((T, hkv, hd), dtype=dt, device="cuda")
    A.qk_norm_rope(q, k, pos, freqs, q_out, k_out=k_out, v=v, k_cache=c[0], v_cache=c[1], slots=slots, k_s=c[2],
                   v_s=c[3], q_w=wq, k_w=wk, eps=1e-6, one_plus=T != 3, sections=sections, interleaved=inter)
    torch.cuda.synchronize()
    axis = _axis(half, sections, inter)
    u = R.half_step(dt)
    sub = 2.0 ** -25 if dt == FP else 0.0
    rq, tq = _ref(q, wq, 1e-6, T != 3, pos, freqs, axis)
    rk, tk = _ref(k, wk, 1e-6, T != 3, pos, freqs, axis)
    R.check(q_out, rq, u * rq.abs() + 1.01 * tq + sub, "queries")
    R.check(k_out, rk, u * rk.abs() + 1.01 * tk + sub, "keys")
    there = (slots >= 0) & (slots < pages * page)
    s = slots[there].long()
    at, off = s // page, s % page
    left = torch.ones((pages, page), dtype=torch.bool, device="cuda")
    left[at, off] = False
    for n, x, x_s, ref, t32 in (("keys", 0, 2, rk, tk), ("values", 1, 3, v.double(), v.double() * 0)):
        assert torch.equal(c[x][left], old[x][left]), n
        ref, t32 = ref[there], t32[there]
        if not int8:
            R.check(c[x][at, off], ref, u * ref.abs() + 1.01 * t32 + sub, "cached " + n)
            continue
        assert torch.equal(c[x_s][left], old[x_s][left]), n
        want = (ref.abs().amax(-1) / 127).clamp_min(1e-8)
        got = c[x_s][at, off].double()
        assert ((got - want).abs() <= want * 2.0 ** -19).all(), n
        R.check(c[x][at, off].double() * got[..., None], ref, 0.5001 * got[..., None] + 1.01 * t32, "codes of " + n)


def test_in_place_without_norm_and_without_cache():
    from qwen35_amd.kernels import attention as A
    q, k, _, g = _inputs(40, 4, 2, 128, BF, 1)
    q0, k0 = q.clone(), k.clone()
    pos = torch.arange(40, device="cuda")
    freqs = torch.tensor([1e4 ** (-i / 64) for i in range(64)], dtype=torch.float32, device="cuda")
    assert A.qk_norm_rope(q, k, pos, freqs, q, k_out=k) is q
    torch.cuda.synchronize()
    for y, x in ((q, q0), (k, k0)):
        ref, t = _ref(x, None, 0, True, pos[None], freqs, [0] * 64)
        R.check(y, ref, R.half_step(BF) * ref.abs() + 1.01 * t)


def test_far_positions_keep_their_angle():
    from qwen35_amd.kernels import attention as A
    q, k, _, g = _inputs(5, 1, 1, 64, FP, 2)
    pos = torch.tensor([0, 2 ** 31 - 1, 2 ** 31, 10 ** 9 + 7, 2 ** 33], device="cuda")
    freqs = torch.ones(32, dtype=torch.float64, device="cuda") * 0.7310585786300049
    out = torch.empty_like(q.contiguous())
    A.qk_norm_rope(q, k, pos, freqs, out, k_out=torch.empty_like(k.contiguous()))
    ref, t = _ref(q, None, 0, True, pos[None], freqs, [0] * 32)
    # the 64-bit angle itself: a product and a difference at up to 6.3e9, 2 * 2^33 * 2^-53
    R.check(out, ref, R.half_step(FP) * ref.abs() + 1.01 * t + 2 ** -18 * q.double().abs().amax())


def test_no_rotation_and_rows_that_hold_no_number():
    from qwen35_amd.kernels import attention as A
    q, k, v, g = _inputs(4, 2, 2, 64, BF, 3)
    k[1, 0, 5] = torch.nan
    v[2, 1, 7] = torch.inf
    c = R.cache(2, 16, 2, 64, BF, 4, True)
    none = torch.empty(0, dtype=torch.float32, device="cuda")
    pos = torch.zeros(4, dtype=torch.int64, device="cuda")
    out = torch.empty((4, 2, 64), dtype=BF, device="cuda")
    w = torch.zeros(64, dtype=BF, device="cuda")
    slots = torch.tensor([3, 9, 20, 31], device="cuda")
    A.qk_norm_rope(q, k, pos, none, out, v=v, k_cache=c[0], v_cache=c[1], slots=slots, k_s=c[2], v_s=c[3], q_w=w, k_w=w)
    torch.cuda.synchronize()
    ref, t = _ref(q, w, 1e-6, True, pos[None], none, [])
    R.check(out, ref, R.half_step(BF) * ref.abs() + t)
    kd, vd = (c[i][slots // 16, slots % 16].double() * c[i + 2][slots // 16, slots % 16][..., None] for i in (0, 1))
    assert kd[1, 0].isnan().all() and kd[1, 1].isfinite().all()
    assert not vd[2, 1].isfinite().all() and vd[2, 0].isfinite().all()


def test_empty():
    from qwen35_amd.kernels import attention as A
    q = torch.empty((0, 2, 64), dtype=BF, device="cuda")
    A.qk_norm_rope(q, q, torch.empty(0, dtype=torch.int64, device="cuda"), torch.ones(8, device="cuda"), q, k_out=q)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("dt", [BF, FP])
def test_codes_of_values_are_the_formulas(hd, dt):
    """Values are not turned: their scales and codes come out bit for bit, ties included."""
    from qwen35_amd.kernels import attention as A
    T, hkv, page = 300, 2, 16
    q, k, v, g = _inputs(T, 4, hkv, hd, dt, 31)
    v = v.clone()
    v[:100, :, 0] = 127 / 64  # scales of a power of two, and values that lie on ties
    v[:100, :, 1:] = torch.randint(-253, 254, (100, hkv, hd - 1), generator=g, device="cuda").to(dt) / 128
    v[100:110] = 0
    pages = -(-T // page)
    kc, vc = (torch.zeros((pages, page, hkv, hd), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, page, hkv), device="cuda") for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    A.qk_norm_rope(q, k, torch.arange(T, device="cuda"), torch.ones(16, device="cuda") * 0.1, torch.empty_like(q), v=v,
                   k_cache=kc, v_cache=vc, slots=slots, k_s=ks, v_s=vs)
    # quotients in 64 bits, rounded (53 bits are more than twice 24 and two: as divided in 32; torch
    # multiplies by the reciprocal of a number)
    x = v.double()
    s = (x.abs().amax(-1) / 127).float().clamp_min(1e-8)
    r = (x / s[..., None].double()).float()
    code = torch.trunc(r + torch.where(r >= 0, 0.5, -0.5)).to(torch.int8)
    assert torch.equal(vs.view(-1, hkv)[slots], s)
    assert torch.equal(vc.view(-1, hkv, hd)[slots], code)
