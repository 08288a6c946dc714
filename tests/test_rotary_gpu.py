"""Rotary positions with gradients on the GPU, against complex numbers in 64 bits."""

import pytest
import torch

from ksanadit_amd import train_ops

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def turned(x, frequencies, positions, sections=None, interleaved=True, magnitude=1.0, sign=1.0):
    """(x's rows turned, the largest value of each pair's: what roundings are relative to), both float64 ``[B, L, H, D]``.  positions: ``[B, L]`` or ``[B, L, axes]``."""
    pairs = frequencies.shape[0]
    axis = [a for a, n in enumerate(sections or (pairs,)) for _ in range(n)]
    at = positions.double()
    at = at[..., axis] if sections is not None else at.unsqueeze(-1).expand(*at.shape, pairs)
    turn = torch.polar(torch.full_like(at, 1.0), sign * at * frequencies)[:, :, None] * magnitude
    x = x.double()
    own, rest = x[..., : 2 * pairs], x[..., 2 * pairs :]
    a, b = (own[..., 0::2], own[..., 1::2]) if interleaved else (own[..., :pairs], own[..., pairs:])
    z = torch.complex(a, b) * turn
    size = (a.abs() + b.abs()) * abs(magnitude)

    def woven(c, d):
        return torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)

    return torch.cat((woven(z.real, z.imag), rest), -1), torch.cat((woven(size, size), torch.zeros_like(rest)), -1)


def check(got, x, frequencies, positions, sections, interleaved, magnitude=1.0, sign=1.0):
    """Off by half a step of the type, and of the pair's size by: the angle's remainder, its factor pi / 2 and their product 0.8 * 3, the series 2, the
    magnitude 1, the two products and their sum 2 halves of an fp32 step - below 8; and by what 64 bits leave of the angle, 2^-51 of it in both."""
    want, size = turned(x, frequencies, positions, sections, interleaved, magnitude, sign)
    far = float((positions.double().abs().max() if positions.numel() else 0.0) * frequencies.max())
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 + size * (8 * 2.0**-24 + far * 2.0**-50) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


CASES = [
    # B, L, H, Hkv, D, width, interleaved, sections, dtype
    (1, 1, 1, 1, 128, 128, True, None, "bf16"),
    (2, 5, 8, 2, 128, 128, False, None, "bf16"),
    (2, 33, 40, 8, 128, 128, True, (22, 21, 21), "fp16"),
    (3, 17, 12, 4, 80, 32, False, None, "fp32"),
    (1, 300, 3, 3, 64, 64, True, None, "fp32"),
    (2, 7, 5, 0, 96, 48, True, (8, 8, 8), "bf16"),
    (2, 7, 5, 1, 96, 48, False, (24, 0), "bf16"),
    (1, 9, 2, 2, 80, 40, False, None, "bf16"),   # halves of 20: value by value
    (1, 9, 2, 2, 80, 20, True, None, "fp16"),
    (2, 11, 3, 1, 7, 6, False, None, "bf16"),    # an odd head
    (2, 11, 3, 1, 7, 2, True, None, "fp32"),
    (1, 4, 70, 70, 72, 8, True, None, "fp16"),   # an odd number of groups of eight
    (1, 3, 2, 2, 512, 512, False, None, "bf16"),
    (1, 3, 2, 2, 510, 256, False, (32, 32, 32, 32), "fp32"),
    (1, 6, 300, 40, 64, 32, False, None, "bf16"),
]


@pytest.mark.parametrize("B,L,H,Hkv,D,width,interleaved,sections,dtype", CASES)
@pytest.mark.parametrize("far", [None, 1000003])
def test_rows_and_gradients(hip_device, B, L, H, Hkv, D, width, interleaved, sections, dtype, far):
    g = torch.Generator(device=hip_device).manual_seed(D + L)
    frequencies = train_ops.rotary_frequencies(width, sections=sections, device=hip_device)
    shape = (B, L) if sections is None else (B, L, len(sections))
    positions = None
    if far or sections:
        positions = torch.randint(-(far or 50), far or 50, shape, generator=g, device=hip_device, dtype=torch.int64 if far else torch.int32)
    rows = [torch.randn((B, L, h, D), generator=g, device=hip_device).to(DTYPES[dtype]).requires_grad_() for h in (H, Hkv) if h]
    grads = [torch.randn(t.shape, generator=g, device=hip_device).to(t.dtype) for t in rows]
    out = train_ops.rotary(*rows, frequencies=frequencies, positions=positions, sections=sections, interleaved=interleaved, magnitude=1.25)
    out = out if isinstance(out, tuple) else (out,)
    back = torch.autograd.grad(out, rows, grads)
    at = torch.arange(L, device=hip_device).expand(B, L) if positions is None else positions
    for x, y, dy, dx in zip(rows, out, grads, back):
        assert y.dtype == x.dtype and y.shape == x.shape
        check(y.detach(), x.detach(), frequencies, at, sections, interleaved, 1.25)
        check(dx, dy, frequencies, at, sections, interleaved, 1.25, -1.0)
    with torch.no_grad():
        again = train_ops.rotary(*rows, frequencies=frequencies, positions=positions, sections=sections, interleaved=interleaved, magnitude=1.25)
    for y, z in zip(out, again if isinstance(again, tuple) else (again,)):
        assert torch.equal(y, z)


@pytest.mark.parametrize("interleaved", [True, False])
def test_channels_behind_the_width_are_copied(hip_device, interleaved):
    """Their bits, whatever stands beside them."""
    x = torch.randn(2, 5, 3, 128, device=hip_device).bfloat16()
    x[0, 0, 0, 32:] = torch.tensor([float("nan"), float("inf"), -0.0, -float("inf")], device=hip_device).repeat(24).bfloat16()
    y = train_ops.rotary(x, frequencies=train_ops.rotary_frequencies(32, device=hip_device), interleaved=interleaved)
    assert torch.equal(y[..., 32:].contiguous().view(torch.int16), x[..., 32:].contiguous().view(torch.int16))
    assert bool(y[..., :32].isfinite().all())


@pytest.mark.parametrize("kind", ["HND", "sliced", "expanded", "odd address", "strided channels"])
def test_layouts(hip_device, kind):
    g = torch.Generator(device=hip_device).manual_seed(3)
    f = train_ops.rotary_frequencies(64, device=hip_device)
    plain = torch.randn((2, 9, 4, 64), generator=g, device=hip_device).half()
    layout, x = "NHD", plain
    if kind == "HND":
        layout, x = "HND", plain.transpose(1, 2).contiguous()
    elif kind == "sliced":
        x = torch.zeros((2, 9, 12, 64), dtype=plain.dtype, device=hip_device)[:, :, 4:8]
        x.copy_(plain)
    elif kind == "expanded":
        plain = plain[:1, :, :1].expand(2, 9, 4, 64)
        x = plain
    elif kind == "odd address":
        x = torch.zeros(plain.numel() + 1, dtype=plain.dtype, device=hip_device)[1:].view(plain.shape)
        x.copy_(plain)
    else:
        x = torch.zeros((2, 9, 4, 128), dtype=plain.dtype, device=hip_device)[..., ::2]
        x.copy_(plain)
    x = x.detach().requires_grad_()
    y = train_ops.rotary(x, frequencies=f, tensor_layout=layout)
    dy = torch.randn((2, 9, 4, 64), generator=g, device=hip_device).half()
    (dx,) = torch.autograd.grad(y, x, dy.transpose(1, 2) if layout == "HND" else dy)
    if layout == "HND":
        y, dx = y.transpose(1, 2), dx.transpose(1, 2)
    at = torch.arange(9, device=hip_device).expand(2, 9)
    check(y.detach(), plain, f, at, None, True)
    check(dx, dy, f, at, None, True, sign=-1.0)


def test_positions_in_their_layouts(hip_device):
    f = train_ops.rotary_frequencies(64, sections=(16, 8, 8), device=hip_device)
    x = torch.randn(3, 10, 2, 64, device=hip_device)
    wide = torch.randint(0, 5000, (3, 20, 6), device=hip_device, dtype=torch.int32)
    for at in (wide[:, ::2, ::2], wide[:1, :10, 3:], wide[1, 10:, :3], wide[:1, :10, 3:].expand(3, 10, 3), wide[:, 3:4, :3].expand(3, 10, 3), wide[:, :10, :1].expand(3, 10, 3)):
        y = train_ops.rotary(x, frequencies=f, positions=at, sections=(16, 8, 8))
        check(y, x, f, at.expand(3, 10, 3), (16, 8, 8), True)
        y = train_ops.rotary(x, frequencies=f, positions=at.long(), sections=(16, 8, 8))
        check(y, x, f, at.expand(3, 10, 3), (16, 8, 8), True)


def test_which_gradients_are_wanted(hip_device):
    f = train_ops.rotary_frequencies(64, device=hip_device)
    q, k = torch.randn(1, 4, 3, 64, device=hip_device, requires_grad=True), torch.randn(1, 4, 2, 64, device=hip_device)
    a, b = train_ops.rotary(q, k, frequencies=f)
    (dq,) = torch.autograd.grad(a.sum() + b.sum(), q)
    check(dq, torch.ones_like(q), f, torch.arange(4, device=hip_device).expand(1, 4), None, True, sign=-1.0)
    k.requires_grad_()
    a, b = train_ops.rotary(q, k, frequencies=f)
    assert torch.autograd.grad(b.sum(), (q, k), allow_unused=True)[0] is None
    assert b.requires_grad and train_ops.rotary(k.detach(), frequencies=f).requires_grad is False


def test_gradients_of_gradients(hip_device):
    """Linear: the gradient of <turn^T dy, w> for dy is w turned."""
    f = train_ops.rotary_frequencies(64, device=hip_device)
    x, dy, w = (torch.randn(2, 4, 3, 64, device=hip_device, requires_grad=True) for _ in range(3))
    (dx,) = torch.autograd.grad(train_ops.rotary(x, frequencies=f), x, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dx, dy, w)
    check(ddy.detach(), w.detach(), f, torch.arange(4, device=hip_device).expand(2, 4), None, True)


def test_differences(hip_device):
    f = train_ops.rotary_frequencies(32, device=hip_device)
    x, d, dy = (torch.randn(1, 3, 2, 32, device=hip_device) for _ in range(3))
    x.requires_grad_()
    (dx,) = torch.autograd.grad(train_ops.rotary(x, frequencies=f, interleaved=False, magnitude=0.5), x, dy)
    with torch.no_grad():
        moved = [train_ops.rotary(x + s * d, frequencies=f, interleaved=False, magnitude=0.5).double() for s in (1, -1)]
    # (a linear map's difference is exact but for fp32: 192 products of numbers below 5 with 2^-22 each)
    assert abs(float(((moved[0] - moved[1]) / 2 * dy.double()).sum() - (dx.double() * d.double()).sum())) < 192 * 25 * 2.0**-22


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ahead_of_the_training_attention(hip_device, dtype):
    """A block's way: norm, rotary, attention, back to the leaves.  The gradients are those of the attention's inputs turned back."""
    g = torch.Generator(device=hip_device).manual_seed(6)
    B, L, H, Hkv, D, sections = 2, 150, 4, 2, 128, (22, 21, 21)
    f = train_ops.rotary_frequencies(D, sections=sections, device=hip_device)
    at = torch.randint(0, 60, (B, L, 3), generator=g, device=hip_device, dtype=torch.int32)
    x = {n: torch.randn((B, L, h * D), generator=g, device=hip_device).to(DTYPES[dtype]).requires_grad_() for n, h in (("q", H), ("k", Hkv))}
    v = torch.randn((B, L, Hkv, D), generator=g, device=hip_device).to(DTYPES[dtype])
    do = torch.randn((B, L, H, D), generator=g, device=hip_device).to(DTYPES[dtype])
    weight = torch.rand(H * D, generator=g, device=hip_device)
    q, k = (train_ops.residual_norm(t, norm="rms", weight=weight[: t.shape[2]])[1].unflatten(2, (-1, D)) for t in x.values())
    qr, kr = train_ops.rotary(q, k, frequencies=f, positions=at, sections=sections)
    o = train_ops.attention(qr, kr, v)
    inner = torch.autograd.grad(o, (qr, kr), do, retain_graph=True)
    outer = torch.autograd.grad(o, (q, k), do, retain_graph=True)
    for dy, dx in zip(inner, outer):
        check(dx, dy, f, at, sections, True, sign=-1.0)
    leaves = torch.autograd.grad(o, tuple(x.values()), do, retain_graph=True)
    again = torch.autograd.grad((q, k), tuple(x.values()), outer)
    assert all(torch.equal(a, b) for a, b in zip(leaves, again))


def test_hooks_may_lay_saved_tensors_out_anew(hip_device):
    f = train_ops.rotary_frequencies(64, sections=(16, 16), device=hip_device)
    at = torch.randint(0, 99, (2, 5, 4), device=hip_device)[..., ::2]
    x = torch.randn(2, 5, 3, 64, device=hip_device, requires_grad=True)
    with torch.autograd.graph.save_on_cpu():
        y = train_ops.rotary(x, frequencies=f, positions=at, sections=(16, 16))
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    check(dx, torch.ones_like(x), f, at, (16, 16), True, sign=-1.0)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.int() if t.dtype == torch.int64 else t, lambda t: t):
        y = train_ops.rotary(x, frequencies=f, positions=at, sections=(16, 16))
    with pytest.raises(RuntimeError, match="hooks"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_streams_and_graphs(hip_device):
    f = train_ops.rotary_frequencies(128, device=hip_device)
    x = torch.randn(2, 64, 8, 128, device=hip_device).bfloat16().requires_grad_()
    at = torch.arange(64, device=hip_device, dtype=torch.int32)
    dy = torch.randn_like(x).detach()

    def step():
        y = train_ops.rotary(x, frequencies=f, positions=at)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for shift in (0, 5, 1000):
        at.copy_(torch.arange(64, device=hip_device) + shift)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_what_records_operators_is_refused(hip_device):
    f = train_ops.rotary_frequencies(64, device=hip_device)
    x = torch.randn(1, 4, 2, 64, device=hip_device)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        train_ops.rotary(torch.autograd.forward_ad.make_dual(x, x), frequencies=f)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.fx.experimental.proxy_tensor.make_fx(lambda x: train_ops.rotary(x, frequencies=f))(x)


def test_a_compiled_function_calls_it(hip_device):
    f = train_ops.rotary_frequencies(64, device=hip_device)
    x = torch.randn(1, 4, 2, 64, device=hip_device, requires_grad=True)
    compiled = torch.compile(lambda x: train_ops.rotary(x * 2, frequencies=f) * 2, backend="aot_eager")
    for _ in range(3):
        y = compiled(x)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        z = train_ops.rotary(x * 2, frequencies=f) * 2
        assert torch.equal(y, z) and torch.equal(dx, torch.autograd.grad(z, x, torch.ones_like(z))[0])


def test_nothing_to_turn(hip_device):
    f = train_ops.rotary_frequencies(64, device=hip_device)
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)):
        x = torch.empty(shape, device=hip_device, requires_grad=True)
        y = train_ops.rotary(x, frequencies=f)
        assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    q, k = torch.randn(1, 4, 2, 64, device=hip_device), torch.empty(1, 4, 0, 64, device=hip_device)
    a, b = train_ops.rotary(q, k, frequencies=f)
    assert b.shape == k.shape
    check(a, q, f, torch.arange(4, device=hip_device).expand(1, 4), None, True)


def test_refusals(hip_device):
    f = train_ops.rotary_frequencies(64, device=hip_device)
    x = torch.randn(2, 4, 3, 64, device=hip_device)
    at = torch.arange(4, device=hip_device)
    for kw, what in (({"frequencies": f.float()}, "float64"), ({"frequencies": f.cpu()}, "device"), ({"frequencies": f.repeat(2)}, "go with heads"),
                     ({"frequencies": f[::2]}, "contiguous"), ({"frequencies": f[:0]}, "go with heads"), ({"frequencies": f.clone().requires_grad_()}, "no gradient"),
                     ({"sections": (16, 8)}, "sections"), ({"sections": (33, -1)}, "negative"), ({"sections": (8, 8, 8, 4, 4)}, "sections"),
                     ({"positions": at.float()}, "positions"), ({"positions": at[:3]}, "positions"), ({"positions": at.cpu()}, "positions"),
                     ({"positions": at[None].expand(3, 4)}, "positions"), ({"positions": at, "sections": (16, 16)}, "positions"),
                     ({"magnitude": float("inf")}, "magnitude"), ({"tensor_layout": "LHD"}, "tensor_layout"), ({"k": x[:1]}, "incompatible"), ({"k": x.half()}, "one type")):
        with pytest.raises(ValueError, match=what):
            train_ops.rotary(x, **{"frequencies": f, **kw})
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        train_ops.rotary(x.double(), frequencies=f)
    with pytest.raises(NotImplementedError, match="512"):
        train_ops.rotary(torch.zeros(1, 1, 1, 514, device=hip_device), frequencies=f)
