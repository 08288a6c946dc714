"""The attention with gradients on the GPU, against its formula in 64 bits.

Tolerances count roundings.  Let u = eps / 2 be the tensors' half step.  A result is rounded once (u of itself); probabilities,
and in the backward pass their gradients and the result in d = rowsum(dO o), are rounded once each where they enter a sum (u of
each term, so at most u times the sum of the terms' absolute values).  fp32 sums of n terms add n 2^-24 of the same absolute sums,
far below u here.  Every bound below is that: factor u |terms| summed, with the absolute sums formed in 64 bits.

fp16 is a fixed-point format below 2^-14: its values are multiples of 2^-24 there, and rounding to nearest is off by up to 2^-25 however
small the value.  That is added once per rounding: to a result as it is; to a probability, which is scaled by 2^15 in the backward
pass and by 2^6 against the row's largest one (at most 1) in the forward pass, 2^-40 and 2^-31; to a gradient of a score, scaled by 2^15
and a power of two of at least half of 1 / (2 max|dO| max|v|), 2^-40 times 4 max|dO| max|v|.  (bf16 has fp32's exponents: nothing.)

dq.  A row's exact dS sum to zero, so c sum dS k = c sum dS (k - m) whatever m is.  The kernel forms c (sum dS' k - (sum dS') m) with its own dS' =
dS + e, which is c sum (dS + e) (k - m): off by c sum e (k - m), so |k - m| stands in the bound where |k| would without m - more for a key that
is smaller than the mean, less where keys share an offset.  m is the mean of the entry's first min(64, count) keys for rows that see them all, and of
what they see for others.  There the sum of dS', which is one of e, goes into a product once more, its share of each key rounded to the tensors' type: u
(and in fp16 the step below 2^-14, scaled as for dS) times the sum of e over the keys' number, on every key.  Sums, the mean and the product with it are fp32: at most 2^-20 of sum |dS| (|k| + |m|) besides.

So much for any kernel with that m, and these bounds stand.  The kernel's own m is nearer to what a row attends to (an estimate of sum P k), for which its first
term, P times what d is off by, nearly vanishes: it keeps to half of them, and ``test_keys_of_two_kinds`` says what it keeps to that a first tile's mean does not."""

import ctypes as C
import math

import pytest
import torch

from ksanadit_amd import _capi, train_ops

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

    qs = abs(scale) * qd.abs()
    # of dq: rows that see all of the entry's first keys, and those that do not
    counts = torch.full((B,), Lk) if k_lens is None else torch.as_tensor(k_lens).clamp(0, Lk)
    first = [min(64, int(n)) for n in counts]
    m = torch.stack([kd[b, :, : max(1, n)].mean(1, keepdim=True) for b, n in enumerate(first)])
    e_dq = e_ds @ (kd - m).abs()
    for b, n in enumerate(first):
        for r in range(min(n - 1, Lq) if causal else 0):  # row r sees keys 0 to r
            own = kd[b, :, : r + 1]
            e = e_ds[b, :, r, : r + 1].unsqueeze(1)
            again = u * e.mean(2, keepdim=True) + (2.0**-40 * most if half else 0.0)
            e_dq[b, :, r] = (e @ (own - own.mean(1, keepdim=True)).abs() + again * own.abs().sum(1, keepdim=True)).squeeze(1)
    e_dq = abs(scale) * (e_dq + 2.0**-20 * (ds.abs() @ (kd.abs() + m.abs())))
    return (*pair(o, e_fwd @ vd.abs() + soft.amax(-1, keepdim=True) * o.abs()), *pair(ds @ kd * scale, e_dq),
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


# ------------------------------------------------------------------------------------------------ scales and magnitudes
@gpu
@pytest.mark.parametrize("scale", [-0.09, 0.0, 1.0])
def test_any_scale(hip_device, scale):
    _check(*_draw(1, 1, 2, 1, 70, 130, 64, torch.float16, std=0.5), hip_device, scale=scale, causal=True)


@gpu
@pytest.mark.parametrize("do_std", [1e-6, 300.0])
def test_gradients_of_any_size_in_fp16(hip_device, do_std):
    """Loss-scaled and vanishing gradients: nothing inside overflows or vanishes that the result can hold."""
    _check(*_draw(2, 1, 2, 2, 150, 400, 128, torch.float16, do_std=do_std), hip_device)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_reference_points_that_move(hip_device, dtype):
    """Scores that grow from tile to tile, by less and by more than the points may lag, and rows that only see small ones."""
    q, k, v, do = _draw(4, 1, 1, 1, 64, 640, 128, dtype)
    k *= (0.2 + torch.arange(640).view(1, -1, 1, 1) / 200).to(dtype)
    _check(q, k, v, do, hip_device, causal=False)


# ------------------------------------------------------------------------------------------------ layouts
def _attend(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = train_ops.attention(*leaves, **kw)
    return (o.detach(), *torch.autograd.grad(o, leaves, do))


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_layouts_give_the_same_bits(hip_device):
    q, k, v, do = (t.to(hip_device) for t in _draw(6, 2, 6, 3, 150, 170, 64, torch.bfloat16))
    want = _attend(q, k, v, do)
    assert _same(_attend(q, k, v, do), want)  # and repeated calls
    # slices of a fused projection, heads before positions, a base that is not aligned, gradients with strides of zero
    fused = torch.empty(2, 170, 12, 64, dtype=q.dtype, device=hip_device)
    fused[:, :150, :6], fused[:, :, 6:9], fused[:, :, 9:] = q, k, v
    assert _same(_attend(fused[:, :150, :6], fused[:, :, 6:9], fused[:, :, 9:], do), want)
    first = [t.transpose(1, 2).contiguous() for t in (q, k, v, do)]
    got = _attend(*first, tensor_layout="HND")
    assert _same([t.transpose(1, 2) for t in got], want)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=hip_device)[1:].view(t.shape).copy_(t) for t in (q, k, v, do)]
    assert _same(_attend(*odd), want)
    ones = torch.ones((), dtype=q.dtype, device=hip_device).expand(do.shape)
    assert _same(_attend(q, k, v, ones), _attend(q, k, v, ones.contiguous()))


@gpu
def test_counts_of_any_kind(hip_device):
    q, k, v, do = (t.to(hip_device) for t in _draw(7, 2, 2, 2, 90, 100, 128, torch.float16))
    want = _attend(q, k, v, do, k_lens=torch.tensor([60, 100], dtype=torch.int32, device=hip_device), q_lens=torch.tensor([90, 33], device=hip_device))
    assert _same(_attend(q, k, v, do, k_lens=[60, 100], q_lens=torch.tensor([90, 33])), want)
    with pytest.raises(ValueError, match="k_lens"):
        train_ops.attention(q, k, v, k_lens=[3])


@gpu
def test_only_wanted_gradients(hip_device):
    q, k, v, do = (t.to(hip_device) for t in _draw(8, 1, 2, 2, 100, 140, 128, torch.bfloat16))
    _, dq, dk, dv = _attend(q, k, v, do)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(train_ops.attention(*leaves), [leaves[i] for i in wanted], do)
        assert _same(got, [(dq, dk, dv)[i] for i in wanted])
    assert not train_ops.attention(q, k, v).requires_grad
    with torch.no_grad():
        assert not train_ops.attention(*[t.detach().requires_grad_() for t in (q, k, v)]).requires_grad


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,Hq,Hkv,Lq,Lk,D,causal", [(1, 8, 8, 700, 300, 128, False), (2, 8, 4, 333, 500, 64, True), (1, 4, 1, 64, 3000, 128, False)])
def test_gradients_of_keys_do_not_hang_on_who_else_wants_one(hip_device, dtype, B, Hq, Hkv, Lq, Lk, D, causal):
    """Rows' numbers come along with dq where that is wanted, and from a kernel of their own where it is not: the same bits, in every row."""
    for seed in range(4):
        q, k, v, do = (t.to(hip_device) for t in _draw(40 + seed, B, Hq, Hkv, Lq, Lk, D, dtype))
        _, _, dk, dv = _attend(q, k, v, do, is_causal=causal)
        leaves = [k.detach().requires_grad_(), v.detach().requires_grad_()]
        assert _same(torch.autograd.grad(train_ops.attention(q, *leaves, is_causal=causal), leaves, do), (dk, dv))


@gpu
def test_saved_tensors_may_be_kept_elsewhere(hip_device):
    q, k, v, do = (t.to(hip_device) for t in _draw(9, 2, 4, 2, 100, 140, 64, torch.bfloat16))
    want = _attend(q, k, v, do, k_lens=[140, 31])
    wide = [torch.zeros(*t.shape[:2], 2 * t.shape[2], t.shape[3], dtype=t.dtype, device=hip_device)[:, :, ::2].copy_(t) for t in (q, k, v)]
    with torch.autograd.graph.save_on_cpu():  # they come back contiguous
        got = _attend(*wide, do, k_lens=[140, 31])
    assert _same(got, want)


@gpu
def test_saved_tensors_may_be_laid_out_anew(hip_device):
    """Statistics and counts too: each comes back with its last dimension a stride of two apart."""
    q, k, v, do = (t.to(hip_device) for t in _draw(10, 2, 4, 2, 100, 140, 64, torch.float16))
    want = _attend(q, k, v, do, k_lens=[140, 31], q_lens=[7, 100])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack((t, torch.full_like(t, 7)), -1)[..., 0]):
        got = _attend(q, k, v, do, k_lens=[140, 31], q_lens=[7, 100])
    assert _same(got, want)


@gpu
@pytest.mark.parametrize("of", ["q", "lse", "lens"])
def test_saved_tensors_left_elsewhere_are_refused(hip_device, of):
    """What a hook gives back on the host is no address that a kernel reads."""
    q = torch.zeros(1, 20, 2, 64, device=hip_device, dtype=torch.float16, requires_grad=True)
    kind = {"q": torch.float16, "lse": torch.float32, "lens": torch.int32}[of]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu() if t.dtype == kind else t):
        o = train_ops.attention(q, q, q, k_lens=torch.tensor([15], dtype=torch.int32, device=hip_device))
    with pytest.raises(RuntimeError, match="came back"):
        o.backward(torch.zeros_like(o))


@gpu
def test_what_cannot_be_differentiated_is_refused(hip_device):
    q = torch.randn(1, 20, 1, 64, device=hip_device, dtype=torch.float16, requires_grad=True)
    lens = torch.tensor([15], dtype=torch.int32, device=hip_device)
    o = train_ops.attention(q, q, q, k_lens=lens)
    (g,) = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)
    o = train_ops.attention(q, q, q, k_lens=lens)
    lens.fill_(3)  # after the forward pass has used it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with pytest.raises(ValueError, match="dtype"):
        train_ops.attention(*[q.float()] * 3)
    with pytest.raises(ValueError, match="one device and one dtype"):
        train_ops.attention(q, q.bfloat16(), q)
    with pytest.raises(NotImplementedError, match="head size"):
        train_ops.attention(*[torch.zeros(1, 4, 1, 96, device=hip_device, dtype=torch.float16)] * 3)
    with pytest.raises(ValueError, match="not a multiple"):
        train_ops.attention(q.expand(1, 20, 3, 64), q.expand(1, 20, 2, 64), q.expand(1, 20, 2, 64))


@gpu
def test_nothing_to_attend_from_or_to(hip_device):
    def t(*shape):
        return torch.randn(shape, device=hip_device, dtype=torch.bfloat16, requires_grad=True)

    for q, k, v in ((t(1, 0, 2, 64), t(1, 5, 2, 64), t(1, 5, 2, 64)), (t(1, 5, 2, 64), t(1, 0, 2, 64), t(1, 0, 2, 64)), (t(0, 5, 2, 64),) * 3):
        o = train_ops.attention(q, k, v)
        assert o.shape == q.shape and not o.any()
        o.sum().backward()
        assert not q.grad.any() and not k.grad.any() and not v.grad.any()


# ------------------------------------------------------------------------------------------------ streams, graphs, sizes
@gpu
def test_streams_and_graphs(hip_device):
    """The same bits from another stream, and from graphs with the backward pass in them: replayed several times with other inputs and
    with eager work between the replays; two graphs side by side share nothing."""
    sets = [[t.to(hip_device) for t in _draw(20 + i, 1, 4, 2, 200, 900, 128, torch.float16)] for i in range(3)]
    want = [_attend(*s, is_causal=True) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert _same(_attend(*sets[0], is_causal=True), want[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        inputs = [torch.empty_like(t) for t in sets[0]]
        for a, b in zip(inputs, sets[0]):
            a.copy_(b)
        with torch.cuda.stream(side):  # (warmed up on the capturing stream, as torch asks)
            side.wait_stream(torch.cuda.current_stream())
            _attend(*inputs, is_causal=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outputs = _attend(*inputs, is_causal=True)
        graphs.append((graph, inputs, outputs))
    for turn in range(4):
        for at, (graph, inputs, outputs) in enumerate(graphs):
            s = (turn + at) % 3
            for a, b in zip(inputs, sets[s]):
                a.copy_(b)
            graph.replay()
            _attend(*sets[(s + 1) % 3])  # eager work of the same kind
            torch.cuda.synchronize()
            assert _same(outputs, want[s])


@gpu
def test_offsets_beyond_32_bits(hip_device):
    """Keys and values of 2.3 billion elements each, by heads of the last batch entry against the formula."""
    B, L, H, D = 2, 70000, 128, 128
    g = torch.Generator(device=hip_device).manual_seed(1)
    k, v = (torch.randn((B, L, H, D), generator=g, device=hip_device, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    q, do = (torch.randn((B, 3, H, D), generator=g, device=hip_device, dtype=torch.bfloat16) for _ in range(2))
    q.requires_grad_()
    assert k.numel() > 2**31
    got = (o := train_ops.attention(q, k, v), *torch.autograd.grad(o, (q, k, v), do))
    for h in (0, H - 1):
        part = [t.detach()[1:, :, h : h + 1].cpu() for t in (q, k, v, do)]
        want = _formula(*part)
        for x, y, most in zip(got, want[::2], want[1::2]):
            assert ((x.detach()[1:, :, h : h + 1].cpu().double() - y).abs() <= most).all()


@gpu
@pytest.mark.parametrize("Hq,Hkv,Lq,Lk,causal", [(16, 4, 1500, 1500, True), (40, 40, 1560, 1560, False), (2, 2, 5000, 77, False), (3, 3, 64, 9000, False)])
def test_cut_loops_against_uncut_ones(hip_device, Hq, Hkv, Lq, Lk, causal):
    """Blocks whose loops are cut into runs, and the same heads among enough others that nothing is cut: results that differ by their
    roundings only, each within what the formula allows."""
    q, k, v, do = _draw(11, 1, Hq, Hkv, Lq, Lk, 128, torch.bfloat16)
    got = _attend(*(t.to(hip_device) for t in (q, k, v, do)), is_causal=causal)
    h, hk = Hq - 1, Hkv - 1
    rep = Hq // Hkv
    part = (q[:, :, h - rep + 1 :], k[:, :, hk:], v[:, :, hk:], do[:, :, h - rep + 1 :])
    want = _formula(*part, causal=causal)
    for x, y, most in zip(got, want[::2], want[1::2]):
        x = x[:, :, -y.shape[2] :].cpu().double()
        assert ((x - y).abs() <= most).all()


@gpu
@pytest.mark.parametrize("Lk", [60, 256, 2048])
def test_keys_whose_scores_leave_the_range_of_fp32(hip_device, Lk):
    """Every eighth key (and with it all that dq estimates the mean key by, of 256 and more) has a score of minus infinity, finite as it is itself: it
    weighs nothing, and the others' gradients are what they are without it, to the roundings of dS and of the result (u each, of sums of a few hundred
    terms in no order: four of their root mean squares)."""
    q, k, v, do = _draw(24, 1, 2, 2, 100, Lk, 128, torch.bfloat16)
    q, k = ((q.float().abs() + 0.1) * 1e19).bfloat16(), (k.float() * 1e-19).bfloat16()
    k[:, ::8] = -1e20
    others = torch.arange(Lk) % 8 != 0
    got = [t.cpu().double() for t in _attend(*(t.to(hip_device) for t in (q, k, v, do)))]
    assert all(t.isfinite().all() for t in got) and not got[2][:, ~others].any() and not got[3][:, ~others].any()
    want, rms = _dq_rms(q, k[:, others], v[:, others], do, False)
    assert (got[1] - want).norm() <= 4 * rms


def _runs_scratch(q, k, causal, k_lens):
    """Bytes that the runs of a call's cut loops need, forward and backward: none where every block is walked whole"""
    lib, n = _capi.load(), (C.c_uint64 * 2)()
    call = train_ops._attention_call(q, k, k, q, causal, None, k_lens, None)
    assert lib.ksana_sage_train_attn_scratch(call, C.addressof(n), C.addressof(n) + 8) == 0
    B, Lq, Hq, _ = q.shape
    Lk, Hkv = k.shape[1:3]
    tiles = -(-Lq * Hq // Hkv // 64)
    rows = 2 * (-(-B * Hkv * tiles * 64 * 4 // 256) * 256) + -(-B * Hkv * (tiles + (-(-Lk // 64) if q.dtype == torch.float16 else 0)) * 4 // 256) * 256
    return n[0], n[1] - rows


@gpu
@pytest.mark.parametrize("B,Hq,Hkv,Lq,Lk,D,dtype,causal,k_lens,copies,forward_too", [
    (1, 4, 4, 1024, 1024, 128, torch.bfloat16, False, None, 16, True), (1, 4, 4, 1024, 1024, 64, torch.float16, False, None, 48, True),
    (1, 4, 2, 1000, 900, 128, torch.bfloat16, True, None, 32, True), (1, 8, 8, 8192, 100, 128, torch.bfloat16, False, None, 64, False),
    (1, 6, 2, 5, 4000, 128, torch.float16, False, None, 256, True), (2, 4, 4, 600, 700, 64, torch.bfloat16, False, [700, 333], 96, True)])
def test_the_same_heads_cut_and_whole(hip_device, B, Hq, Hkv, Lq, Lk, D, dtype, causal, k_lens, copies, forward_too):
    """Few heads, whose loops are cut into runs (of the keys alone where queries are many), and copies of them that fill the card, none of which is."""
    t = _draw(23, B, Hq, Hkv, Lq, Lk, D, dtype)
    want = _formula(*t, causal=causal, k_lens=k_lens)
    for n in (1, copies):
        q, k, v, do = (x.to(hip_device).repeat(n, 1, 1, 1) for x in t)
        lens = None if k_lens is None else torch.tensor(k_lens * n, dtype=torch.int32, device=hip_device)
        fwd, bwd = _runs_scratch(q, k, causal, lens)
        assert (fwd > 0, bwd > 0) == (n == 1 and forward_too, n == 1)
        got = _attend(q, k, v, do, is_causal=causal, k_lens=lens)
        for name, x, y, most in zip(("o", "dq", "dk", "dv"), got, want[::2], want[1::2]):
            assert torch.equal(x[:B], x[-B:]), name
            off = ((x[:B].cpu().double() - y).abs() / most).max().item()
            assert off <= 1.0, f"{name}: {off:.2f} of what roundings allow, {n} copies"


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,Hq,Hkv,Lq,Lk,D,causal,k_lens", [
    (1, 2, 2, 300, 700, 128, False, None), (1, 4, 2, 300, 300, 64, True, None), (1, 6, 2, 5, 4000, 128, False, None), (2, 2, 2, 150, 200, 128, True, [200, 33])])
def test_keys_that_share_an_offset(hip_device, dtype, B, Hq, Hkv, Lq, Lk, D, causal, k_lens):
    """Off zero by eight times what they vary: the bound of dq, which counts |k - m|, knows nothing of it."""
    q, k, v, do = _draw(17, B, Hq, Hkv, Lq, Lk, D, dtype)
    off = 8 * torch.randn((1, 1, Hkv, D), generator=torch.Generator().manual_seed(18))
    _check(q * 0.25, (k.float() + off).to(dtype), v, do, hip_device, causal=causal, k_lens=k_lens)


def _kinds(seed, dtype, Hq, Hkv, Lq, Lk, D, first, attended):
    """Keys of which the first ones are off the others by four times what these vary, and queries that lean to one kind or to neither"""
    q, k, v, do = _draw(seed, 1, Hq, Hkv, Lq, Lk, D, dtype)
    off = torch.randn((1, 1, Hkv, D), generator=torch.Generator().manual_seed(seed + 1))
    k = torch.cat((k[:, :first].float() + 4 * off, k[:, first:].float()), 1).to(dtype)
    return (q.float() + 0.5 * attended * off.repeat_interleave(Hq // Hkv, 2)).to(dtype), k, v, do


def _dq_rms(q, k, v, do, causal):
    """dq in 64 bits and the root of the sum of squares that its roundings leave, whatever keys are there.

    The kernel forms c sum (dS + e) (k - m).  e holds each dS' rounding, of variance at most u^2 / 3 dS^2, and P times what d is off by, whose sum
    over P (k - m) vanishes where m is the row's own mean key sum P k.  So with it the variance is at most c^2 sum u^2 / 3 dS^2 |k - m|^2, plus u^2 / 3 dq^2 for
    the result.  d is off by the roundings of o (dO^2 o^2) and of P (P^2 dP^2), in sum of about twice the variance of e without it (o^2 has the size of sum P^2 in
    each channel, dP^2 that of |dO|^2): with m from a sample, that is by |m' - m|^2 <= |k - m|^2 off, at most 1 + 2 + 1 times the variance.  (fp16: 2^-40 of
    4 max|dO| max|v| at most besides, its values' spacing, and 2^-25 of a result.)"""
    B, Lq, Hq, D = q.shape
    rep, u = Hq // k.shape[2], HALF_STEP[q.dtype]
    qd, dod = (t.double().transpose(1, 2) for t in (q, do))
    kd, vd = (t.double().transpose(1, 2).repeat_interleave(rep, 1) for t in (k, v))
    s = qd @ kd.transpose(2, 3) * D**-0.5
    if causal:
        s = s.masked_fill(torch.ones(s.shape[2:], dtype=torch.bool).triu(1), -math.inf)
    p = s.softmax(-1)
    dp = dod @ vd.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    mean = p @ kd
    spread = (kd * kd).sum(-1).unsqueeze(2) - 2 * mean @ kd.transpose(2, 3) + (mean * mean).sum(-1, keepdim=True)  # |k - m|^2
    half = q.dtype == torch.float16
    fixed = 2.0**-40 * 4 * dod.norm(dim=-1).max() * vd.norm(dim=-1).max() if half else 0.0
    dq = ds @ kd * D**-0.5
    variance = ((u * u / 3 * ds * ds + fixed**2 * (p > 0)) * spread).sum() / D + u * u / 3 * (dq * dq).sum() + (2.0**-50 * dq.numel() if half else 0.0)
    return dq.transpose(1, 2), variance.sqrt()


_KINDS = [  # Hq, Hkv, Lq, Lk, D, of the first kind, queries lean to it, causal
    (2, 2, 300, 1024, 128, 64, -1, False), (4, 2, 200, 1000, 64, 500, -1, False), (4, 2, 200, 1000, 128, 500, 1, False), (2, 2, 150, 2000, 128, 250, 0, False),
    (2, 1, 100, 9000, 128, 64, -1, False), (2, 2, 800, 800, 128, 400, -1, True), (2, 2, 30, 40, 64, 20, -1, False)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,Lq,Lk,D,first,attended,causal", _KINDS)
def test_keys_of_two_kinds(hip_device, dtype, Hq, Hkv, Lq, Lk, D, first, attended, causal):
    """A few keys in front or half of them off the others, as text in front of an image: twice (four times the variance) what roundings leave."""
    t = _kinds(19, dtype, Hq, Hkv, Lq, Lk, D, first, attended)
    want, rms = _dq_rms(*t, causal)
    got = _attend(*(x.to(hip_device) for x in t), is_causal=causal)[1].cpu().double()
    off = ((got - want).norm() / rms).item()
    assert off <= 2.0, f"dq {off:.2f} times what roundings leave (relative error {((got - want).norm() / want.norm()).item():.5f})"


@gpu
@pytest.mark.parametrize("B,Hq,Hkv,Lq,Lk,D,dtype,k_lens,q_lens", [
    (1, 8, 2, 1500, 1500, 64, torch.bfloat16, None, None), (2, 6, 2, 600, 2300, 64, torch.float16, None, None), (1, 5, 1, 1900, 700, 128, torch.bfloat16, None, None),
    (1, 3, 1, 40, 9000, 128, torch.float16, None, None), (4, 48, 48, 290, 290, 128, torch.bfloat16, None, None),
    (4, 48, 16, 290, 270, 64, torch.float16, [270, 0, 131, 64], [290, 5, 129, 1]), (2, 4, 4, 200, 6000, 64, torch.bfloat16, [6000, 77], None)])
def test_causal_blocks_whole_and_in_runs(hip_device, B, Hq, Hkv, Lq, Lk, D, dtype, k_lens, q_lens):
    """Blocks of which later ones see more: more of them than the card holds at once, and few, with runs that some do not have."""
    _check(*_draw(13, B, Hq, Hkv, Lq, Lk, D, dtype), hip_device, causal=True, k_lens=k_lens, q_lens=q_lens)


# ------------------------------------------------------------------------------------------------ where the package offers it
@gpu
def test_the_backend_trains_where_it_is_asked_to(hip_device):
    from ksanadit_amd import KsanaAttentionBackend, KsanaAttentionConfig
    from ksanadit_amd.backends.sage_attn import SageAttentionImpl

    q, k, v, do = (t.to(hip_device) for t in _draw(12, 1, 2, 2, 100, 120, 128, torch.bfloat16))
    make = lambda **kw: SageAttentionImpl(KsanaAttentionConfig(backend=KsanaAttentionBackend.SAGE_ATTN), 2, 128, False, 128**-0.5, **kw)  # noqa: E731
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = make(trainable=True).forward(*leaves)
    assert _same((o.detach(), *torch.autograd.grad(o, leaves, do)), _attend(q, k, v, do))
    assert torch.equal(make(trainable=True).forward(q, k, v), make().forward(q, k, v))  # without gradients: as ever
    assert make(trainable=True, out_dtype=torch.float16).forward(*leaves).dtype == torch.float16


@gpu
@pytest.mark.parametrize("causal", [False, True])
def test_the_op_trains_where_it_is_asked_to(hip_device, causal):
    from ksanadit_amd import KsanaAttentionConfig, pick_attn_op

    q, k, v, do = (t.to(hip_device) for t in _draw(21, 1, 4, 2, 100, 120, 128, torch.bfloat16))
    make = pick_attn_op(KsanaAttentionConfig(backend="sage_attention"))
    op, plain = (make(num_heads=4, head_size=128, num_kv_heads=2, causal=causal, **kw) for kw in ({"trainable": True}, {}))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = op(*leaves)
    assert _same((o.detach(), *torch.autograd.grad(o, leaves, do)), _attend(q, k, v, do, is_causal=causal))
    assert torch.equal(op(q, k, v), plain(q, k, v))  # without gradients: the quantized attention, as ever
    leaves = [t.float().requires_grad_() for t in (q, k, v)]  # (cast to bf16, as for the quantized attention)
    o = op(*leaves)
    assert o.dtype == torch.float32 and _same([t.bfloat16() for t in torch.autograd.grad(o, leaves, do.float())], _attend(q, k, v, do, is_causal=causal)[1:])


@gpu
def test_a_compiled_function_calls_it(hip_device):
    """The kernels are no operators of torch: a compiled function leaves its graph for them, in the forward and the backward pass, in every call."""
    q, k, v, do = (t.to(hip_device) for t in _draw(22, 1, 2, 2, 60, 70, 64, torch.bfloat16))
    f = torch.compile(lambda q, k, v: train_ops.attention(q * 2, k, v) * 2, backend="aot_eager")
    for scale in (1, 3):
        leaves = [(t * scale).requires_grad_() for t in (q, k, v)]
        o = f(*leaves)
        got = (o.detach(), *torch.autograd.grad(o, leaves, do))
        want = _attend(leaves[0].detach() * 2, leaves[1].detach(), leaves[2].detach(), do * 2)
        assert _same(got, (want[0] * 2, want[1] * 2, *want[2:]))
