"""The operators with gradients where no GPU is needed: what they refuse, and the tests' own formulas against differences."""

import ctypes as C
import weakref

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from ksanadit_amd import _capi, train_ops
from tests.test_train_attention_gpu import HALF_STEP, _draw, _formula
from tests.test_train_norm_gpu import ALL, definition, make


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype)


# ------------------------------------------------------------------------------------------------ the formulas
def _directional(f, inputs, directions, step):
    plus, minus = (f([x + sign * step * d for x, d in zip(inputs, directions)]) for sign in (1, -1))
    return (plus - minus) / (2 * step)


@pytest.mark.parametrize("causal,lens", [(False, None), (True, None), (True, ([5, 0], [9, 7]))])
def test_the_attention_formula_against_differences(causal, lens):
    """Central differences of sum(o * do): off by step^2 / 6 times a third derivative (below 1e3 for these sizes) and 2^-52 / step."""
    k_lens, q_lens = lens if lens else (None, None)
    q, k, v, do = _draw(3, 2, 4, 2, 9, 11, 8, torch.float32)
    HALF_STEP[torch.float64] = 0.0
    try:
        q, k, v, do = (t.double() for t in (q, k, v, do))
        kw = dict(causal=causal, k_lens=k_lens, q_lens=q_lens)
        o, _, dq, _, dk, _, dv, _ = _formula(q, k, v, do, **kw)
        g = torch.Generator().manual_seed(1)
        directions = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (q, k, v)]
        got = _directional(lambda x: (_formula(*x, do, **kw)[0] * do).sum(), (q, k, v), directions, 1e-5)
    finally:
        del HALF_STEP[torch.float64]
    want = sum((a * b).sum() for a, b in zip((dq, dk, dv), directions))
    assert abs(got - want) <= 1e-6 * max(1.0, abs(want))


@pytest.mark.parametrize("norm,post,names", [("layer", None, ALL[:4]), ("rms", "layer", ALL), ("layer", "rms", ALL), ("rms", None, ("weight",))])
def test_the_norm_definition_against_differences(norm, post, names):
    t, dh, dn = make(2, 2, 5, 12, torch.float32, torch.float32, torch.float32, names)
    t = {k: v.double() for k, v in t.items()}
    dh, dn = dh.double() * ("y" in names), dn.double()
    r = 0.7 if "y" in names else 1.0
    full = definition(t, dh, dn, norm, post, r, 1e-6)
    g = torch.Generator().manual_seed(1)
    directions = [torch.randn(v.shape, generator=g, dtype=torch.float64) for v in t.values()]

    def value(x):
        d = definition(dict(zip(t, x)), dh, dn, norm, post, r, 1e-6)
        return (d["h"][0] * dh).sum() + (d["n"][0] * dn).sum()

    got = _directional(value, list(t.values()), directions, 1e-5)
    want = sum((full[k][0] * d).sum() for k, d in zip(t, directions))
    assert abs(got - want) <= 1e-6 * max(1.0, abs(want))


# ------------------------------------------------------------------------------------------------ refusals
def test_tensors_off_the_gpu_are_refused():
    q = _meta(1, 4, 2, 64)
    with pytest.raises(RuntimeError, match="HIP device"):
        train_ops.attention(q, q, q)
    with pytest.raises(RuntimeError, match="HIP device"):
        train_ops.residual_norm(_meta(1, 4, 64))


def test_arguments_of_the_attention():
    q = _meta(1, 4, 2, 64)
    with pytest.raises(ValueError, match="4-D"):
        train_ops.attention(q[0], q, q)
    with pytest.raises(ValueError, match="tensor_layout"):
        train_ops.attention(q, q, q, tensor_layout="LHD")


def test_arguments_of_the_norm():
    x = _meta(2, 4, 64)
    for kw, what in (({"norm": "batch"}, "unknown"), ({"post_norm": "l2", "y": x}, "unknown"), ({"y": x[:, :3]}, "one shape")):
        with pytest.raises(ValueError, match=what):
            train_ops.residual_norm(x, **kw)
    with pytest.raises(ValueError, match="one shape"):
        train_ops.residual_norm(x[0])
    for name, shape in (("gate", (3, 64)), ("weight", (2, 64)), ("shift", (2, 4, 64)), ("scale", (63,))):
        with pytest.raises(ValueError, match=name):
            train_ops._norm_vector(name, torch.empty(shape), x)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        train_ops._norm_vector("gate", torch.empty(64, dtype=torch.float64), x)


def _attn_call(**kw):
    B, Hq, Hkv, Lq, Lk, D = (kw.pop(n, d) for n, d in zip(("B", "Hq", "Hkv", "Lq", "Lk", "D"), (1, 4, 2, 16, 16, 128)))

    def strides(L, H):
        return _capi.Strides(L * H * D, H * D, D, 1)

    c = _capi.TrainAttn(_capi.Shape(B, Hq, Hkv, Lq, Lk, D), 0, 0, 0.1, 0, strides(Lq, Hq), strides(Lk, Hkv), strides(Lk, Hkv), strides(Lq, Hq), None, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw,rc", [
    ({}, 0), ({"B": 0}, -1), ({"Hkv": 3}, -1), ({"D": 96}, -2), ({"Lk": 0}, -1), ({"dtype": 2}, -1), ({"reserved": 1}, -1), ({"sm_scale": float("inf")}, -1),
    ({"sm_scale": float("nan")}, -1), ({"Lq": 1 << 25}, -2), ({"Lk": (1 << 24) + 1}, -2), ({"Hq": 8192, "Hkv": 1, "Lq": 1 << 10}, -2),
    ({"Hq": 70000, "Hkv": 70000}, -2), ({"q_lens": 2}, -1), ({"k_lens": 3}, -1), ({"B": 1024, "Hq": 60, "Hkv": 60, "Lk": 1 << 20}, -2)])
def test_calls_of_the_attention_are_checked(kw, rc):
    lib, n = _capi.load(), C.c_uint64(0)
    assert lib.ksana_sage_train_attn_scratch(C.addressof(_attn_call(**kw)), C.addressof(n), C.addressof(n)) == rc, lib.ksana_sage_last_error()
    assert lib.ksana_sage_train_attn_scratch(None, None, None) == -1


def test_cut_loops_stay_within_a_launch():
    """Workgroups of a launch, 256 threads each, as the scratch of the runs tells them: fewer than 2^24, whatever is asked for."""
    lib, g = _capi.load(), torch.Generator().manual_seed(3)
    n, cut = C.c_uint64(0), 0
    for _ in range(4000):
        B, heads, group, Lq, Lk = (int(2 ** (torch.rand((), generator=g) * bits)) for bits in (10, 9, 4, 24, 24))
        c = _attn_call(B=B, Hq=heads * group, Hkv=heads, Lq=Lq, Lk=Lk, D=64 * int(torch.randint(1, 3, (), generator=g)), causal=int(torch.randint(2, (), generator=g)))
        if lib.ksana_sage_train_attn_scratch(C.addressof(c), C.addressof(n), None) == 0:
            workgroups = n.value // (128 * (c.shape.D + 2) * 4)  # cut blocks times their runs
            assert workgroups < 2**24
            cut += workgroups > 0
    assert cut > 500


@pytest.mark.parametrize("change,what", [
    (dict(q=None), b"q is null"), (dict(k=0x1008), b"not 16-byte"), (dict(lse=0x1002), b"lse"), (dict(c=dict(q_strides=_capi.Strides(1, 2, 3, 1))), b"stride"),
    (dict(c=dict(v_strides=_capi.Strides(4096, 256, 128, 2))), b"D stride"), (dict(scratch=None), b"scratch is null"), (dict(scratch=0x1010), b"256-byte"),
    (dict(c=dict(k_strides=_capi.Strides(1 << 40, 1 << 33, 128, 1))), b"beyond"),
    (dict(bwd=True, dk=None), b"together"), (dict(bwd=True, dq=0x1008), b"gradient"), (dict(bwd=True, lse=None), b"lse"), (dict(bwd=True, do=None), b"d_o is null")])
def test_buffers_of_the_attention_are_checked(change, what):
    """Nothing here reaches a device: the library looks at addresses, never through them."""
    lib = _capi.load()
    # (keys for many runs, so that scratch is needed)
    c = _attn_call(Lk=4096, **change.get("c", {}))
    a = {n: 0x1000 for n in ("q", "k", "v", "o", "lse", "scratch", "do", "dq", "dk", "dv")}
    a.update({k: v for k, v in change.items() if k in a})
    if change.get("bwd"):
        st = _capi.Strides(*c.q_strides)
        rc = lib.ksana_sage_train_attn_bwd(C.addressof(c), a["q"], a["k"], a["v"], a["o"], a["lse"], a["do"], C.addressof(st), a["dq"], a["dk"], a["dv"],
                                           a["scratch"], None)
    else:
        rc = lib.ksana_sage_train_attn_fwd(C.addressof(c), a["q"], a["k"], a["v"], a["o"], a["lse"], a["scratch"], None)
    assert rc in (-1, -2) and what in lib.ksana_sage_last_error(), lib.ksana_sage_last_error()


def _norm_call(vectors=None, **kw):
    v = {n: _capi.Vector() for n in train_ops._VECTORS} | (vectors or {})
    d = dict(B=2, L=3, C=64, x_dtype=0, y_dtype=0, norm=1, post=0, residual_scale=1.0, eps=1e-6, reserved=0) | kw
    return _capi.TrainNorm(*d.values(), (C.c_int64 * 2)(192, 64), (C.c_int64 * 2)(192, 64), *v.values())


@pytest.mark.parametrize("kw,rc,what", [
    ({"C": 8193}, -2, b"8192"), ({"L": 0}, -1, b"extent"), ({"x_dtype": 0, "y_dtype": 1}, -1, b"types"), ({"x_dtype": 3}, -1, b"types"), ({"norm": 0}, -1, b"norm"),
    ({"norm": 3}, -1, b"norm"), ({"post": -1}, -1, b"post"), ({"eps": -1.0}, -1, b"eps"), ({"eps": float("nan")}, -1, b"eps"), ({"reserved": 5}, -1, b"reserved"),
    ({"vectors": {"post_weight": _capi.Vector(0x1000, 0, 2, 0)}}, -1, b"post_weight"), ({"vectors": {"gate": _capi.Vector(0x1000, 0, 5, 0)}}, -1, b"dtype"),
    ({"vectors": {"weight": _capi.Vector(0x1000, 64, 2, 0)}}, -1, b"batch stride"), ({"vectors": {"shift": _capi.Vector(0x1001, 0, 0, 0)}}, -1, b"aligned")])
def test_calls_of_the_norm_are_checked(kw, rc, what):
    lib = _capi.load()
    assert lib.ksana_sage_train_norm_fwd(C.addressof(_norm_call(**kw)), 0x1000, 0x1000, 0x1000, 0x1000, None, None) == rc
    assert what in lib.ksana_sage_last_error()


def test_buffers_of_the_norm_are_checked():
    lib, call = _capi.load(), _norm_call()
    good = C.addressof(call)
    fwd = lib.ksana_sage_train_norm_fwd
    assert fwd(good, None, 0x1000, 0x1000, 0x1000, None, None) == -1 and b"x is null" in lib.ksana_sage_last_error()
    assert fwd(good, 0x1000, 0x1000, None, 0x1000, None, None) == -1 and b"h is null" in lib.ksana_sage_last_error()
    assert fwd(good, 0x1001, 0x1000, 0x1000, 0x1000, None, None) == -1
    scaled = _norm_call(residual_scale=0.5)
    assert fwd(C.addressof(scaled), 0x1000, None, None, 0x1000, None, None) == -1 and b"go with y" in lib.ksana_sage_last_error()
    grads = (C.c_void_p * 6)(None, 0x1000, None, None, None, None)
    bwd = lib.ksana_sage_train_norm_bwd
    assert bwd(good, 0x1000, 0x1000, 0x1000, None, 0x1000, 0x1000, 0x1000, C.addressof(grads), 0x1000, None) == -1 and b"absent" in lib.ksana_sage_last_error()
    none = (C.c_void_p * 6)()
    assert bwd(good, 0x1000, 0x1000, 0x1000, None, 0x1000, 0x1000, None, C.addressof(none), 0x1000, None) == -1 and b"dy" in lib.ksana_sage_last_error()
    assert bwd(good, 0x1000, 0x1000, 0x1000, None, 0x1000, 0x1000, 0x1000, C.addressof(none), None, None) == -1 and b"scratch" in lib.ksana_sage_last_error()


def test_packed_structures_are_the_librarys():
    """Byte by byte what the ctypes structures hold."""
    q, k = torch.empty(2, 7, 6, 64, dtype=torch.float16), torch.empty(2, 9, 3, 128, dtype=torch.float16)[..., :64]
    lens = torch.zeros(2, dtype=torch.int32)
    c = _capi.TrainAttn(_capi.Shape(2, 6, 3, 7, 9, 64), 1, 1, 0.25, 0, *(_capi.Strides(*t.stride()) for t in (q, k, k, q)), None, lens.data_ptr())
    assert bytes(c) == train_ops._attention_call(q, k, k, q, True, 0.25, lens, None)
    x, g, w = torch.empty(2, 5, 48), torch.empty(2, 3, 48, dtype=torch.bfloat16)[:, 1:2], torch.empty(48, dtype=torch.float16)
    none = _capi.Vector()
    n = _capi.TrainNorm(2, 5, 48, 2, 0, 2, 1, 0.5, 1e-5, 0, (C.c_int64 * 2)(240, 48), (C.c_int64 * 2)(240, 48), _capi.Vector(g.data_ptr(), 144, 0, 0), none, none,
                        _capi.Vector(w.data_ptr(), 0, 1, 0), none, none)
    assert bytes(n) == train_ops._norm_call(x, x.bfloat16(), [g, None, None, w, None, None], "rms", "layer", 0.5, 1e-5, torch.bfloat16)


def test_scales_that_fp32_cannot_hold(monkeypatch):
    monkeypatch.setattr(train_ops, "_check_attention", lambda *a: None)
    q = _meta(1, 4, 2, 64)
    for scale in (float("nan"), float("inf"), -1e39):
        with pytest.raises(ValueError, match="sm_scale"):
            train_ops.attention(q, q, q, sm_scale=scale)


def _forward_dual(f, t):
    with torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("wants_gradient", [False, True])
@pytest.mark.parametrize("through", [
    _forward_dual, lambda f, t: torch.func.jvp(f, (t,), (t,)), lambda f, t: torch.jit.trace(f, t, check_trace=False), lambda f, t: make_fx(f)(t),
    lambda f, t: make_fx(f, tracing_mode="symbolic")(t), lambda f, t: make_fx(f, pre_dispatch=True)(t)],
    ids=["dual", "jvp", "jit", "fx", "fx_symbolic", "fx_pre_dispatch"])
def test_what_goes_past_the_kernels_is_refused(monkeypatch, on_the_cpu, through, wants_gradient):
    """Forward mode and tracing see torch's own operators only: the result would be without its tangent, the trace without the kernels."""
    on_the_cpu(lambda *a: 0, lambda *a: 0)
    monkeypatch.setattr(train_ops, "_require_hip", lambda *t: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    q, x, w = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 16), torch.zeros(16)
    train_ops.attention(q, q, q)
    train_ops.residual_norm(x)
    for f, t in ((lambda t: train_ops.attention(t, q, q), q), (lambda t: train_ops.attention(q, q, t), q), (lambda t: train_ops.residual_norm(t)[1], x),
                 (lambda t: train_ops.residual_norm(x, t)[0], x), (lambda t: train_ops.residual_norm(x, bias=t)[1], w)):
        with pytest.raises(NotImplementedError, match="forward-mode|cannot be traced"):
            through(f, t.clone().requires_grad_(wants_gradient))


@pytest.mark.parametrize("through", [_forward_dual, lambda f, t: make_fx(f)(t)], ids=["dual", "fx"])
def test_backward_passes_that_go_past_the_kernels_are_refused(on_the_cpu, through):
    on_the_cpu(lambda *a: 0, lambda *a: 0)
    q, x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16, requires_grad=True), torch.zeros(1, 4, 16, requires_grad=True)
    o = train_ops._Attention.apply(q, q, q, False, None, None, None)
    h, n = train_ops._ResidualNorm.apply(x, x, *[None] * 6, "layer", None, 1.0, 1e-6, torch.float32)
    for out, leaf in ((o, q), (h, x), (n, x)):
        torch.autograd.grad(out, leaf, torch.zeros_like(out), retain_graph=True)
        with pytest.raises(NotImplementedError, match="forward-mode|cannot be traced"):
            through(lambda t: torch.autograd.grad(out, leaf, t, retain_graph=True), torch.zeros_like(out))


def test_gradients_of_gradients_are_refused_however_they_are_asked_for(on_the_cpu):
    """With respect to the tensors and to the results' gradients, by which ``torch.autograd.functional.jvp`` gets at a forward derivative."""
    on_the_cpu(lambda *a: 0, lambda *a: 0)
    attend = lambda q: train_ops._Attention.apply(q, q, q, False, None, None, None)  # noqa: E731
    norm = lambda w: train_ops._ResidualNorm.apply(x, x, None, w, None, None, None, None, "layer", None, 1.0, 1e-6, torch.float32)  # noqa: E731
    x = torch.zeros(1, 4, 16)
    for f, t in ((attend, torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)), (norm, torch.zeros(16))):
        with pytest.raises(RuntimeError, match="gradients of gradients"):
            torch.autograd.functional.jvp(f, t, torch.ones_like(t))
        leaf = t.clone().requires_grad_()
        out = f(leaf)
        outs = out if isinstance(out, tuple) else (out,)
        dos = [torch.zeros_like(o).requires_grad_() for o in outs]
        (d,) = torch.autograd.grad(outs, leaf, dos, create_graph=True)
        assert d.shape == leaf.shape and train_ops._not_twice((None, None), leaf) == (None, None)
        for other in (leaf, *dos):
            with pytest.raises(RuntimeError, match="gradients of gradients"):
                torch.autograd.grad(d.sum(), other, retain_graph=True)


# ------------------------------------------------------------------------------------------------ saved tensors that hooks lay out anew
class _Library:
    """Stands for the compiled library on tensors of the CPU: forward passes write what is given, backward passes are looked at."""

    def __init__(self, fwd, bwd):
        self.ksana_sage_train_attn_fwd = self.ksana_sage_train_norm_fwd = fwd
        self.ksana_sage_train_attn_bwd = self.ksana_sage_train_norm_bwd = bwd

    def ksana_sage_train_attn_scratch(self, *a):
        return 0

    def ksana_sage_train_norm_scratch(self, *a):
        return 0


def _memory(address, dtype, n):
    return torch.frombuffer((C.c_char * (n * dtype.itemsize)).from_address(address), dtype=dtype).clone()


def _write(address, t):
    C.memmove(address, t.data_ptr(), t.numel() * t.element_size())


def _laid_out_anew(t):
    """The same values a stride of two apart"""
    return t if t.dim() == 0 else torch.stack((t, torch.full_like(t, 7)), -1)[..., 0]


@pytest.fixture
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(train_ops, "_on", lambda device: train_ops.nullcontext())
    monkeypatch.setattr(train_ops, "_stream_ptr", lambda device: 0)
    return lambda *functions: monkeypatch.setattr(train_ops._capi, "load", lambda: _Library(*functions))


def test_vectors_that_hooks_lay_out_anew(monkeypatch, on_the_cpu):
    """The backward call reads the vectors that the forward pass saved, from memory that nothing else has been given meanwhile."""
    B, L, Ch = 2, 3, 16
    x, y = torch.randn(B, L, Ch), torch.randn(B, L, Ch)
    vectors = [torch.randn(B, 1, Ch) for _ in range(3)] + [torch.randn(Ch) for _ in range(3)]
    copies, seen = [], []
    rows = train_ops._vector_rows

    def watched(t):
        out = rows(t)
        copies.append(weakref.ref(out))
        return out

    monkeypatch.setattr(train_ops, "_vector_rows", watched)

    def bwd(call, *a):
        seen.append(all(c() is not None for c in copies))
        fields = train_ops._NORM.unpack(call)[14:]
        for i, t in enumerate(vectors):
            at, stride = fields[4 * i : 4 * i + 2]
            for b in range(B if t.dim() > 1 else 1):
                seen.append(torch.equal(_memory(at + 4 * b * stride, torch.float32, Ch), t[b, 0] if t.dim() > 1 else t))
        return 0

    on_the_cpu(lambda *a: 0, bwd)
    leaves = [t.requires_grad_() for t in (x, y, *vectors)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _laid_out_anew):
        h, n = train_ops._ResidualNorm.apply(*leaves, "layer", "rms", 1.0, 1e-6, torch.float32)
    torch.autograd.grad((h, n), leaves, (torch.zeros_like(h), torch.zeros_like(n)))
    assert len(copies) == 6 and len(seen) == 1 + 3 * B + 3 and all(seen), seen


def test_a_norms_statistics_that_hooks_lay_out_anew(on_the_cpu):
    stats, seen = torch.randn(2, 3, 4), []

    def fwd(call, x, y, h, n, stats_at, stream):
        _write(stats_at, stats)
        return 0

    def bwd(call, x, y, stats_at, *a):
        seen.append(torch.equal(_memory(stats_at, torch.float32, stats.numel()), stats.flatten()))
        return 0

    on_the_cpu(fwd, bwd)
    x = torch.randn(2, 3, 16, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _laid_out_anew):
        h, n = train_ops._ResidualNorm.apply(x, x, *[None] * 6, "layer", None, 1.0, 1e-6, torch.float32)
    torch.autograd.grad((h, n), x, (torch.zeros_like(h), torch.zeros_like(n)))
    assert seen == [True]


def test_statistics_and_counts_that_hooks_lay_out_anew(on_the_cpu):
    B, Lq, H, D = 2, 5, 3, 64
    q = torch.randn(B, Lq, H, D).bfloat16()
    lse, lens, seen = torch.randn(B, H, Lq), [torch.tensor([4, 5], dtype=torch.int32), torch.tensor([3, 1], dtype=torch.int32)], []

    def fwd(call, q, k, v, o, lse_at, *a):
        _write(lse_at, lse)
        return 0

    def bwd(call, q, k, v, o, lse_at, *a):
        q_lens, k_lens = train_ops._ATTENTION.unpack(call)[-2:]
        seen.extend((torch.equal(_memory(lse_at, torch.float32, lse.numel()), lse.flatten()), torch.equal(_memory(k_lens, torch.int32, B), lens[0]),
                     torch.equal(_memory(q_lens, torch.int32, B), lens[1])))
        return 0

    on_the_cpu(fwd, bwd)
    leaf = q.requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _laid_out_anew):
        o = train_ops._Attention.apply(leaf, leaf, leaf, False, None, *lens)
    torch.autograd.grad(o, leaf, torch.zeros_like(o))
    assert seen == [True] * 3


def test_saved_tensors_that_hooks_make_others_of_are_refused(on_the_cpu):
    on_the_cpu(lambda *a: 0, lambda *a: pytest.fail("called"))
    for change in (lambda t: t.half() if t.dtype == torch.float32 else t, lambda t: t[:1], lambda t: t.long() if t.dtype == torch.int32 else t):
        q = torch.zeros(2, 5, 3, 64, dtype=torch.bfloat16, requires_grad=True)
        x, w = torch.zeros(2, 3, 16, requires_grad=True), torch.zeros(2, 16, requires_grad=True)
        lens = torch.tensor([4, 5], dtype=torch.int32)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            o = train_ops._Attention.apply(q, q, q, False, None, lens, None)
            h, n = train_ops._ResidualNorm.apply(x, x, None, w, None, None, None, None, "layer", None, 1.0, 1e-6, torch.float32)
        with pytest.raises(RuntimeError, match="came back"):
            torch.autograd.grad(o, q, torch.zeros_like(o))
        if change(torch.zeros(2, dtype=torch.int32)).dtype == torch.int32:
            with pytest.raises(RuntimeError, match="came back"):
                torch.autograd.grad((h, n), (x, w), (torch.zeros_like(h), torch.zeros_like(n)))


# ------------------------------------------------------------------------------------------------ through the attention op
def test_the_op_takes_trainable(monkeypatch):
    """torch's SDPA trains as it is (here the backend that a CPU has); a backend that has no backward pass is refused."""
    from ksanadit_amd import KsanaAttentionBackend, KsanaAttentionConfig, attention_op, pick_attn_op
    from ksanadit_amd.backends.radial_sage_attn import RadialSageAttentionImpl

    make = pick_attn_op(KsanaAttentionConfig(backend=KsanaAttentionBackend.TORCH_SDPA))
    q = torch.randn(1, 5, 2, 64, requires_grad=True)
    (g,) = torch.autograd.grad(make(num_heads=2, head_size=64, trainable=True)(q, q, q).square().sum(), q)
    assert g.abs().max() > 0
    monkeypatch.setattr(attention_op, "get_attention_backend_impl", lambda **kw: RadialSageAttentionImpl)
    with pytest.raises(ValueError, match="no backward pass"):
        make(num_heads=2, head_size=64, trainable=True)(q, q, q)


def test_scales_whose_product_with_log2_e_fp32_cannot_hold(monkeypatch):
    """Scores are scaled by sm_scale log2(e): infinite, it made not-a-numbers of scores of zero."""
    monkeypatch.setattr(train_ops, "_check_attention", lambda *a: None)
    q, lib, n = _meta(1, 4, 2, 64), _capi.load(), C.c_uint64(0)
    for scale, rc in ((2.4e38, -1), (-3.3e38, -1), (1.9e38, 0), (-1.9e38, 0)):
        assert lib.ksana_sage_train_attn_scratch(C.addressof(_attn_call(sm_scale=scale)), C.addressof(n), C.addressof(n)) == rc
        if rc != 0:
            with pytest.raises(ValueError, match="sm_scale"):
                train_ops.attention(q, q, q, sm_scale=scale)
