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


def _same(a, b):
    return a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)


@gpu
def test_layouts_give_the_same_bits(hip_device):
    t, dh, dn = make(3, 2, 40, 264, bf16, bf16, fp32, ALL)
    want = _run(t, dh, dn, hip_device, "layer", "rms", 0.5)
    assert _same(_run(t, dh, dn, hip_device, "layer", "rms", 0.5), want)

    def apart(x):  # every other row, column and entry of something larger, at an odd address
        big = torch.zeros([2 * n for n in x.shape[:-1]] + [x.shape[-1] + 3], dtype=x.dtype, device=x.device)
        view = big[tuple(slice(None, None, 2) for _ in x.shape[:-1])][..., 1 : x.shape[-1] + 1]
        return view.copy_(x).detach()

    assert _same(_run(t, dh, dn, hip_device, "layer", "rms", 0.5, wrap=apart), want)
    # a chunk of a modulation table, vectors without their middle dimension, a tensor whose rows are one row
    table = torch.stack([t["gate"], t["scale"], t["shift"]], 1).flatten(1, 2).to(hip_device)
    u = {k: v.to(hip_device) for k, v in t.items()}
    h, n = train_ops.residual_norm(**{**u, "gate": table[:, :1], "scale": table[:, 1:2], "shift": table[:, 2]}, norm="layer", post_norm="rms",
                                   residual_scale=0.5)
    assert torch.equal(h, want["h"]) and torch.equal(n, want["n"])
    row = u["x"][:, :1].expand(-1, 40, -1)
    got, ref = (train_ops.residual_norm(x, u["y"]) for x in (row, row.contiguous()))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@gpu
def test_only_some_results_or_gradients_are_wanted(hip_device):
    t, dh, dn = make(4, 2, 30, 520, fp32, bf16, fp32, ALL)
    u = {k: v.to(hip_device) for k, v in t.items()}
    full = _run(t, dh, dn, hip_device, "rms", "layer", 1.0)
    none = {k: v.double() for k, v in t.items()}
    for use in ("h", "n"):
        leaves = {k: v.clone().requires_grad_() for k, v in u.items()}
        h, n = train_ops.residual_norm(**leaves, norm="rms", post_norm="layer")
        d = torch.autograd.grad(h if use == "h" else n, list(leaves.values()), (dh if use == "h" else dn).to(hip_device), allow_unused=True)
        want = definition(none, dh.double() * (use == "h"), dn.double() * (use == "n"), "rms", "layer", 1.0, 1e-6)
        _check(dict(zip(leaves, d)), want, _types(t, dn))
    leaves = {k: v.clone().requires_grad_(k in ("gate", "weight")) for k, v in u.items()}
    h, n = train_ops.residual_norm(**leaves, norm="rms", post_norm="layer")
    d = torch.autograd.grad((h, n), (leaves["gate"], leaves["weight"]), (dh.to(hip_device), dn.to(hip_device)))
    assert torch.equal(d[0], full["gate"]) and torch.equal(d[1], full["weight"])
    with torch.no_grad():
        h, n = train_ops.residual_norm(**u, norm="rms", post_norm="layer")
    assert torch.equal(h, full["h"]) and torch.equal(n, full["n"])


@gpu
def test_saved_tensors_may_be_kept_elsewhere(hip_device):
    t, dh, dn = make(5, 2, 30, 128, bf16, bf16, bf16, ALL)
    want = _run(t, dh, dn, hip_device, "layer", "layer", 1.0)
    wide = lambda x: torch.zeros(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype, device=x.device)[..., : x.shape[-1]].copy_(x)  # noqa: E731
    with torch.autograd.graph.save_on_cpu():
        assert _same(_run(t, dh, dn, hip_device, "layer", "layer", 1.0, wrap=wide), want)


@gpu
def test_rows_far_from_zero_keep_their_variance(hip_device):
    """Values around 1e4 that differ by 1: squares minus the squared mean would lose them."""
    x = (1e4 + torch.randn(1, 3, 4096, generator=torch.Generator().manual_seed(1))).float()
    t, zero = {"x": x}, torch.zeros_like(x)
    want = definition({"x": x.double()}, zero.double(), zero.double(), "layer", None, 1.0, 1e-6)
    h, n = train_ops.residual_norm(x.to(hip_device))
    assert h.data_ptr() and h.shape == x.shape
    _check({"n": n}, want, _types(t, zero))


@gpu
def test_refusals_and_empty_tensors(hip_device):
    x = torch.randn(2, 3, 16, device=hip_device)
    with pytest.raises(ValueError, match="go with y"):
        train_ops.residual_norm(x, gate=x[0, 0])
    with pytest.raises(ValueError, match="post_weight"):
        train_ops.residual_norm(x, x, post_weight=x[0, 0])
    with pytest.raises(ValueError, match="does not go with"):
        train_ops.residual_norm(x.half(), x)
    with pytest.raises(ValueError, match="its type"):
        train_ops.residual_norm(x, x, out_dtype=torch.float16)
    with pytest.raises(NotImplementedError, match="8192"):
        train_ops.residual_norm(torch.zeros(1, 1, 8200, device=hip_device))
    for shape in ((0, 3, 16), (2, 0, 16)):
        e, w = torch.zeros(shape, device=hip_device, requires_grad=True), torch.ones(16, device=hip_device, requires_grad=True)
        h, n = train_ops.residual_norm(e, e, weight=w)
        (h.sum() + n.sum()).backward()
        assert n.shape == shape and e.grad.shape == shape and not w.grad.any()
    y = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(train_ops.residual_norm(y)[1].square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu
def test_streams_and_graphs(hip_device):
    sets = [make(30 + i, 2, 64, 776, bf16, bf16, fp32, ALL) for i in range(3)]
    want = [_run(*s, hip_device, "layer", "rms", 1.0) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held = {k: v.to(hip_device) for k, v in sets[0][0].items()}
    grads = [g.to(hip_device) for g in sets[0][1:]]

    def step():
        leaves = {k: v.detach().requires_grad_() for k, v in held.items()}
        h, n = train_ops.residual_norm(**leaves, norm="layer", post_norm="rms")
        return {"h": h.detach(), "n": n.detach(), **dict(zip(leaves, torch.autograd.grad((h, n), list(leaves.values()), grads)))}

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert _same(step(), want[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for turn in range(5):
        t, dh, dn = sets[turn % 3]
        for name, v in t.items():
            held[name].copy_(v)
        grads[0].copy_(dh)
        grads[1].copy_(dn)
        graph.replay()
        torch.cuda.synchronize()
        assert _same(out, want[turn % 3])
        _run(*sets[(turn + 1) % 3], hip_device, "rms", "layer", 0.5)  # eager work of the same kind


@gpu
def test_saved_tensors_may_be_laid_out_anew(hip_device):
    """.. with channels a stride of two apart: each is copied, and the copies stay while the kernels read them."""
    t, dh, dn = make(6, 2, 30, 264, bf16, bf16, fp32, ALL)
    want = _run(t, dh, dn, hip_device, "rms", "layer", 0.5)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: torch.stack((x, torch.full_like(x, 7)), -1)[..., 0]):
        got = _run(t, dh, dn, hip_device, "rms", "layer", 0.5)
    assert _same(got, want)


@gpu
@pytest.mark.parametrize("of", [bf16, fp32, fp16], ids=["rows", "statistics", "vectors"])
def test_saved_tensors_left_elsewhere_are_refused(hip_device, of):
    x, w = torch.zeros(2, 3, 16, device=hip_device, dtype=bf16, requires_grad=True), torch.ones(16, device=hip_device, dtype=fp16, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu() if t.dtype == of else t):
        h, n = train_ops.residual_norm(x, x, weight=w)
    with pytest.raises((RuntimeError, ValueError), match="came back|weight must be"):
        torch.autograd.grad((h, n), (x, w), (torch.zeros_like(h), torch.zeros_like(n)))
