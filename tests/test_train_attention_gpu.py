"""The attention with gradients on the GPU, against its formula in 64 bits.

Tolerances count roundings.  Let u = eps / 2 be the tensors' half step.  A result is rounded once (u of itself); probabilities,
and in the backward pass their gradients and the result in d = rowsum(dO o), are rounded once each where they enter a sum (u of
each term, so at most u times the sum of the terms' absolute values).  fp32 sums of n terms add n 2^-24 of the same absolute sums,
far below u here.  Every bound below is that: factor u |terms| summed, with the absolute sums formed in 64 bits.

fp16 is a fixed-point format below 2^-14: its values are multiples of 2^-24 there, and rounding to nearest is off by up to 2^-25 however
small the value.  That is added once per rounding: to a result as it is; to a probability, which is scaled by 2^15 in the backward
pass and by 2^6 against the row's largest one (at most 1) in the forward pass, 2^-40 and 2^-31; to a gradient of a score, scaled by 2^15
and a power of two of at least half of 1 / (2 max|dO| max|v|), 2^-40 times 4 max|dO| max|v|.  (bf16 has fp32's exponents: nothing.)"""

import math

import pytest
import torch

from ksanadit_amd import train_ops

gpu = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _draw(seed, B, Hq, Hkv, Lq, Lk, D, dtype, std=1.0, do_std=1.0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, s=1.0):
        return (torch.randn(shape, generator=g) * s).to(dtype)

    return t(B, Lq, Hq, D, s=std), t(B, Lk, Hkv, D, s=std), t(B, Lk, Hkv, D), t(B, Lq, Hq, D, s=do_std)


def _formula(q, k, v, do, *, causal=False, scale=None, k_lens=None, q_lens=None):
    """Result and gradients in 64 bits, and for each the bound that the roundings leave, [B, L, H, D]."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    u = HALF_STEP[q.dtype]
    scale = D**-0.5 if scale is None else scale
    rep = Hq // Hkv
    qd, dod = (t.double().permute(0, 2, 1, 3) for t in (q, do))
    kd, vd = (t.double().permute(0, 2, 1, 3).repeat_interleave(rep, 1) for t in (k, v))
    seen = torch.ones(B, 1, Lq, Lk, dtype=torch.bool)
    if causal:
        seen &= torch.ones(Lq, Lk, dtype=torch.bool).tril()
    if k_lens is not None:
        seen &= (torch.arange(Lk) < torch.as_tensor(k_lens).view(B, 1)).view(B, 1, 1, Lk)
    if q_lens is not None:
        seen &= (torch.arange(Lq) < torch.as_tensor(q_lens).view(B, 1)).view(B, 1, Lq, 1)
    kd, vd = (torch.where(seen.any(2).unsqueeze(-1), t, 0.0) for t in (kd, vd))  # (what no row sees is not read)
    qd, dod = (torch.where(seen.any(3).unsqueeze(-1), t, 0.0) for t in (qd, dod))
    s = (qd @ kd.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    lse = s.logsumexp(-1, keepdim=True)
    p = torch.where(seen, (s - lse.nan_to_num(neginf=0.0)).exp(), 0.0)
    o = p @ vd
    dp = dod @ vd.transpose(2, 3)
    d = (dod * o).sum(-1, keepdim=True)
    ds = p * (dp - d)
    # d is formed from the rounded result: off by u |dO| |o| summed, on every term of the row
    off = u * (dod.abs() * o.abs()).sum(-1, keepdim=True)
    # the exponent's fp32 rounding: |s| and |lse| 2^-23 each, relative in p
    soft = 2.0**-22 * (s.masked_fill(~seen, 0.0).abs() + lse.nan_to_num(neginf=0.0).abs() + 1)
    half = q.dtype == torch.float16
    e_fwd = p * (u + soft) + (2.0**-31 if half else 0.0) * seen
    e_p = p * (u + soft) + (2.0**-40 if half else 0.0) * seen
    most = 4 * dod.norm(dim=-1).max() * vd.norm(dim=-1).max()
    e_ds = (2.0**-40 * most if half else 0.0) * seen + p * off + ds.abs() * (u + soft) + p * (dp.abs() + d.abs()) * soft + 2.0**-20 * p * (dod.abs() @ vd.abs().transpose(2, 3))

    def heads(t):  # gradients of shared heads are sums
        return t.view(B, Hkv, rep, *t.shape[2:]).sum(2)

    def pair(value, error):
        return value.permute(0, 2, 1, 3), (error + u * value.abs()).permute(0, 2, 1, 3) * 1.01 + (2.0**-25 if half else 1e-30)

    ks, qs = abs(scale) * kd.abs(), abs(scale) * qd.abs()
    return (*pair(o, e_fwd @ vd.abs() + soft.amax(-1, keepdim=True) * o.abs()), *pair(ds @ kd * scale, e_ds @ ks),
            *pair(heads(ds.transpose(2, 3) @ qd) * scale, heads(e_ds.transpose(2, 3) @ qs)),
            *pair(heads(p.transpose(2, 3) @ dod), heads(e_p.transpose(2, 3) @ dod.abs())))


def _check(q, k, v, do, device, **kw):
    want = _formula(q, k, v, do, **kw)
    leaves = [t.to(device).requires_grad_() for t in (q, k, v)]
    o = train_ops.attention(*leaves, is_causal=kw.get("causal", False), sm_scale=kw.get("scale"), k_lens=kw.get("k_lens"), q_lens=kw.get("q_lens"))
    got = (o, *torch.autograd.grad(o, leaves, do.to(device)))
    for name, x, (y, most) in zip(("o", "dq", "dk", "dv"), got, zip(want[::2], want[1::2])):
        x = x.detach().cpu().double()
        assert x.isfinite().all(), name
        off = ((x - y).abs() / most).max().item()
        assert off <= 1.0, f"{name}: {off:.2f} of what roundings allow (largest difference {(x - y).abs().max():.3e})"
    return got


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,Hq,Hkv,Lq,Lk,D,causal", [
    (1, 1, 1, 1, 2, 128, False), (1, 2, 2, 1, 1, 128, False), (2, 2, 1, 33, 31, 128, False), (1, 3, 3, 64, 64, 128, True),
    (1, 2, 2, 128, 64, 64, False), (2, 4, 2, 65, 129, 64, True), (1, 2, 2, 257, 300, 128, False), (1, 2, 2, 300, 257, 128, True),
    (1, 6, 2, 100, 321, 128, True), (1, 5, 1, 77, 200, 128, False), (1, 1, 1, 1, 1000, 128, False), (1, 8, 1, 1, 777, 64, False),
    (1, 260, 260, 70, 66, 128, False), (2, 264, 132, 129, 65, 64, True), (1, 1, 1, 900, 3, 128, False), (1, 2, 2, 513, 513, 128, True), (3, 1, 1, 130, 190, 128, False),
])
def test_result_and_gradients_follow_the_formula(hip_device, dtype, B, Hq, Hkv, Lq, Lk, D, causal):
    _check(*_draw(Lq * 1000 + Lk, B, Hq, Hkv, Lq, Lk, D, dtype), hip_device, causal=causal)


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("k_lens,q_lens", [([0, 70, 200], None), ([200, 1, 64], [1, 130, 0]), (None, [130, 0, 65]), ([-5, 1 << 30, 3], [7, -1, 1 << 30])])
def test_counts_of_padded_batches(hip_device, k_lens, q_lens, causal):
    q, k, v, do = _draw(5, 3, 4, 2, 130, 200, 128, torch.bfloat16)
    for b in range(3):  # what lies behind the counts is never looked at
        if k_lens is not None:
            k[b, max(0, k_lens[b]):] = v[b, max(0, k_lens[b]):] = math.nan
        if q_lens is not None:
            q[b, max(0, q_lens[b]):] = do[b, max(0, q_lens[b]):] = math.nan
    o, dq, dk, dv = _check(q, k, v, do, hip_device, causal=causal, k_lens=k_lens, q_lens=q_lens)
    for b in range(3):
        if k_lens is not None:
            n = max(0, k_lens[b])
            assert not dk[b, n:].any() and not dv[b, n:].any()
        if q_lens is not None:
            n = max(0, q_lens[b])
            assert not o[b, n:].any() and not dq[b, n:].any()
