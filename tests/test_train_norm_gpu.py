"""The gated residual norm with gradients on the GPU, against its definition in 64 bits.

Tolerances count roundings.  A result is rounded once to its type (half a step, u).  Before that everything is fp32: one operation is off by
2^-24 of its result, a sum over the C channels passes through at most 16 additions of a thread, 6 of a wave and 8 of the waves, 2^-19 of
the sum of the absolute terms with all that is multiplied into it, and a sum over rows through at most 128 additions in the
sizes below, 2^-17.  The bounds carry these through the formulas in 64 bits, term by term."""

import pytest
import torch

from ksanadit_amd import train_ops

gpu = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
SMALLEST = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150}  # half of the smallest step
ONE, ROW, COLUMN = 2.0**-22, 2.0**-19, 2.0**-17
VECTORS = ("gate", "scale", "shift", "weight", "bias", "post_weight")


def _normed(t, e, kind, eps):
    """(value, factor, error of the value) of a normalised row whose elements are off by e"""
    mean = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[..., :1])
    centred = t - mean
    inv = (centred.square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = centred * inv
    e_mean = (e.mean(-1, keepdim=True) + ROW * t.abs().mean(-1, keepdim=True)) if kind == "layer" else 0.0
    # the factor is off, relatively, by half of what the mean square is off
    e_inv = (hat.abs() * inv * (e + e_mean)).mean(-1, keepdim=True) + ROW
    return hat, inv, inv * (e + e_mean) + hat.abs() * (e_inv + ONE)


def _back(m, e_m, hat, e_hat, inv, kind):
    """(value, error) of the norm's derivative applied to m"""
    along = (m * hat).mean(-1, keepdim=True)
    e_along = (m.abs() * e_hat + e_m * hat.abs()).mean(-1, keepdim=True) + ROW * (m * hat).abs().mean(-1, keepdim=True)
    mean = m.mean(-1, keepdim=True) if kind == "layer" else 0.0
    e_mean = e_m.mean(-1, keepdim=True) + ROW * m.abs().mean(-1, keepdim=True) if kind == "layer" else 0.0
    inner = m - mean - hat * along
    size = m.abs() + abs(mean) + (hat * along).abs()
    e_inv = (hat.abs() * e_hat).mean(-1, keepdim=True) + ROW
    return inv * inner, inv * (e_m + e_mean + e_hat * along.abs() + hat.abs() * e_along + ONE * size) + inv * inner.abs() * (e_inv + ONE)


def definition(t, dh, dn, norm, post, r, eps):
    """{name: (value, error before the last rounding)}; t: the inputs by name, [B, L, C] and vectors, all in 64 bits"""
    def vec(name, default):
        v = t.get(name)
        return torch.full((1, 1, 1), default, dtype=torch.float64) if v is None else v.reshape(-1, 1, v.shape[-1]) if v.dim() < 3 else v

    x, y = t["x"], t.get("y")
    gate, scale, shift, w, bias, wp = (vec(n, d) for n, d in zip(VECTORS, (1.0, 0.0, 0.0, 1.0, 0.0, 1.0)))
    zero = torch.zeros_like(x)
    if y is None:
        h, e_h, y_hat, e_y, y_inv = x, zero, zero, zero, None
    else:
        y_hat, y_inv, e_y = (y, None, zero) if post is None else _normed(y, zero, post, eps)
        h = r * x + gate * wp * y_hat
        e_h = ONE * ((r * x).abs() + (gate * wp * y_hat).abs()) + (gate * wp).abs() * e_y
    hat, inv, e_hat = _normed(h, e_h, norm, eps)
    a, shifted = w * (1 + scale), bias * (1 + scale) + shift
    out = {"h": (h, e_h), "n": (hat * a + shifted, a.abs() * e_hat + ONE * ((hat * a).abs() + (bias * (1 + scale)).abs() + shift.abs()))}
    m = dn * a
    back, e_back = _back(m, ONE * m.abs(), hat, e_hat, inv, norm)
    d = dh + back
    e_d = e_back + ONE * (dh.abs() + back.abs())
    out["x"] = (r * d, abs(r) * e_d + ONE * (r * d).abs())
    if y is not None:
        through = d * gate * wp
        e_through = (gate * wp).abs() * e_d + ONE * through.abs()
        out["y"] = (through, e_through) if post is None else _back(through, e_through, y_hat, e_y, y_inv, post)

    def over(term, error, dims):
        return term.sum(dims), error.sum(dims) + COLUMN * term.abs().sum(dims)

    def like(name, term, error):
        v = t.get(name)
        if v is None:
            return
        dims = (0, 1) if v.dim() == 1 or v.shape[0] == 1 else (1,)
        value, off = over(term, error, dims)
        out[name] = (value.reshape(v.shape), off.reshape(v.shape))

    like("gate", d * y_hat * wp, (e_d * y_hat.abs() + d.abs() * e_y) * wp.abs())
    like("scale", dn * (hat * w + bias), dn.abs() * e_hat * w.abs() + ONE * dn.abs() * ((hat * w).abs() + bias.abs()))
    like("shift", dn + zero, zero)
    like("weight", dn * (1 + scale) * hat, (dn * (1 + scale)).abs() * e_hat)
    like("bias", dn * (1 + scale), zero)
    like("post_weight", d * gate * y_hat, (e_d * y_hat.abs() + d.abs() * e_y) * gate.abs())
    return out


def make(seed, B, L, C, xt, yt, vt, names, shared=False):
    g = torch.Generator().manual_seed(seed)

    def n(*shape, std=1.0, mean=0.0):
        return mean + std * torch.randn(shape, generator=g)

    t = {"x": n(B, L, C, std=3.0, mean=0.5).to(xt)}
    if "y" in names:
        t["y"] = n(B, L, C).to(yt)
    for name in VECTORS:
        if name in names:
            own = name in ("gate", "scale", "shift") and not shared
            t[name] = n(*((B, 1, C) if own else (C,)), std=0.3, mean=1.0 if "weight" in name else 0.4 if name == "gate" else 0.0).to(vt)
    return t, n(B, L, C).to(xt), n(B, L, C).to(yt)


ALL = ("y",) + VECTORS
bf16, fp16, fp32 = torch.bfloat16, torch.float16, torch.float32


def _check(got, want, types):
    for name, value in got.items():
        y, e = want[name]
        most = 1.01 * (e + HALF_STEP[types[name]] * y.abs()) + SMALLEST[types[name]]
        assert value.dtype == types[name] and value.shape == y.shape, name
        off = (value.detach().cpu().double() - y).abs()
        assert off.isfinite().all(), name
        assert (off <= most).all(), f"{name}: {(off / most).max():.2f} of what roundings allow"


def _run(t, dh, dn, device, norm, post, r, eps=1e-6, wrap=lambda x: x):
    leaves = {k: wrap(v.to(device)).requires_grad_() for k, v in t.items()}
    h, n = train_ops.residual_norm(**leaves, norm=norm, post_norm=post, residual_scale=r, eps=eps, out_dtype=None if "y" in t else dn.dtype)
    outs, grads = ((h, n), (dh, dn)) if "y" in t else ((n,), (dn,))
    d = torch.autograd.grad(outs, list(leaves.values()), [g.to(device) for g in grads])
    return {**({"h": h} if "y" in t else {}), "n": n, **dict(zip(leaves, d))}


def _types(t, dn):
    return {"h": t["x"].dtype, "n": dn.dtype, **{k: v.dtype for k, v in t.items()}}


@gpu
@pytest.mark.parametrize("B,L,C,xt,yt,vt,norm,post,names", [
    (1, 1, 8, bf16, bf16, fp32, "layer", None, ALL[:4]), (1, 1, 1, fp32, fp32, fp32, "rms", "rms", ALL),
    (2, 3, 64, fp16, fp16, fp16, "rms", "rms", ALL), (3, 7, 512, bf16, bf16, bf16, "layer", "layer", ALL),
    (1, 130, 520, fp32, bf16, fp32, "layer", "rms", ALL), (2, 65, 1153, fp16, fp16, fp32, "rms", "layer", ALL),
    (2, 300, 1000, fp32, fp32, fp32, "layer", "layer", ALL), (1, 40, 4096, bf16, bf16, fp32, "rms", None, ("y", "gate", "weight")),
    (2, 33, 5120, bf16, bf16, fp32, "layer", None, ALL[:4]), (1, 9, 8192, fp32, fp16, bf16, "layer", "rms", ALL),
    (1, 5, 8191, bf16, bf16, bf16, "layer", "layer", ALL), (2, 17, 77, fp32, bf16, fp16, "rms", None, ("y",)),
    (1, 12, 200, bf16, bf16, fp32, "layer", None, ("scale", "shift")), (2, 600, 96, fp32, fp16, fp32, "rms", None, ("weight",)),
    (4, 1, 2048, fp32, fp32, fp32, "rms", None, ("y", "scale", "weight")),
])
def test_results_and_gradients_follow_the_definition(hip_device, B, L, C, xt, yt, vt, norm, post, names):
    r = 1.0 if "y" not in names else 0.75
    t, dh, dn = make(B * 10000 + L + C, B, L, C, xt, yt, vt, names)
    want = definition({k: v.double() for k, v in t.items()}, dh.double() if "y" in names else 0.0 * dh.double(), dn.double(), norm, post, r, 1e-6)
    _check(_run(t, dh, dn, hip_device, norm, post, r), want, _types(t, dn))


@gpu
def test_vectors_for_all_entries_sum_their_gradients(hip_device):
    t, dh, dn = make(1, 3, 50, 264, bf16, bf16, fp32, ALL, shared=True)
    want = definition({k: v.double() for k, v in t.items()}, dh.double(), dn.double(), "layer", "rms", 1.0, 1e-6)
    _check(_run(t, dh, dn, hip_device, "layer", "rms", 1.0), want, _types(t, dn))
