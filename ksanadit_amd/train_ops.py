"""Operators with gradients: what a block's attention half needs where it is trained, next to ``sage_ops`` that generates.

``attention`` takes the place of ``sageattn`` where gradients are wanted: the same layouts, key and query counts and causal
masking, 16-bit products without quantization, and a backward pass that recomputes the probabilities.
``residual_norm`` is what stands between two parts of a block: gate, residual sum, norm and modulation in one pass.
``rotary`` gives q and k their rotary positions ahead of the attention.

They run on the tensors' HIP device, on torch's current stream there; scratch comes from torch's caching allocator.  They do not synchronise and may be
captured into a graph, with counts, if any, as int32 tensors on that device (others are copied there in the call, which waits for the copy and cannot be captured).
Repeated calls give the same bits.  Gradients of gradients (``rotary``, which is linear, has them), forward-mode derivatives and tracing are refused; ``torch.compile`` leaves its graph for them.
"""

from __future__ import annotations

import ctypes as C
import struct
from contextlib import nullcontext

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _capi
from .sage_ops import _DTYPES, _k_lens_arg, _require_hip, _stream_ptr, _usable


_HERE = nullcontext()


def _on(device: torch.device):
    """The device made current where it is not: kernels start on the current one.  (Asked for without the detour through torch.cuda, which costs autograd's thread 4 us.)"""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _refuse_unseen(name: str, *tensors: torch.Tensor | None) -> None:
    """The kernels are started past torch's dispatcher: what records its operators, or carries tangents through them, would go on with memory that nothing
    has been written to, or without the tangent."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative (a dual tensor was given)")
    if torch._C._get_tracing_state() is not None or get_proxy_mode() is not None:
        raise NotImplementedError(f"{name} cannot be traced (torch.jit.trace, make_fx): its kernels are not operators of torch")


def _readable(t: torch.Tensor) -> torch.Tensor:
    """The tensor as the kernels read it (``_usable``), a contiguous one at an address that 16 does not divide included."""
    if t.is_contiguous() and t.shape[3] % 8 == 0 and t.data_ptr() % 16 == 0:  # (looking at strides costs more than a kernel of few tokens leaves)
        return t
    t = _usable(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _contiguous_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() and not t.has_names() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _scratch(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _kept(t: torch.Tensor | None, dtype: torch.dtype, shape, device: int) -> torch.Tensor | None:
    """What a forward pass saved for the kernels, contiguous and at an address they read: hooks that keep saved tensors elsewhere may give them back laid
    out and placed otherwise, but not as other tensors."""
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device:
        raise RuntimeError(f"a saved tensor came back from its hooks as {t.dtype} {tuple(t.shape)} on {t.device}, it was {dtype} {tuple(shape)}")
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


# The library's structures, packed (ctypes takes three times as long to build one; a call of few tokens costs what its host work does)
_ATTENTION = struct.Struct("=8ifi16q2Q")  # ksana_sage_train_attn
_NORM = struct.Struct("=7i2fi4q" + 6 * "Qqii")  # ksana_sage_train_norm
_STRIDES, _POINTERS = struct.Struct("=4q"), struct.Struct("=6Q")


def _attention_call(q, k, v, o, is_causal: bool, sm_scale: float | None, k_lens, q_lens) -> bytes:
    B, Lq, Hq, D = q.shape
    return _ATTENTION.pack(B, Hq, k.shape[2], Lq, k.shape[1], D, _DTYPES[q.dtype], is_causal, D**-0.5 if sm_scale is None else sm_scale, 0,
                           *q.stride(), *k.stride(), *v.stride(), *o.stride(), 0 if q_lens is None else q_lens.data_ptr(),
                           0 if k_lens is None else k_lens.data_ptr())


def _check_attention(q, k, v) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention expects 4-D tensors")
    _require_hip(q, k, v)
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"incompatible shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")


def _attention_forward(q, k, v, is_causal, sm_scale, k_lens, q_lens, want_lse: bool):
    """(o, lse or None, bytes of the backward pass's scratch) of ``[B, L, H, D]`` tensors the kernels can read."""
    B, Lq, Hq, D = q.shape
    o = _contiguous_like(q)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=q.device) if want_lse else None
    if q.numel() == 0 or k.numel() == 0:
        return o.zero_(), None if lse is None else lse.fill_(-torch.inf), 0
    lib, call = _capi.load(), _attention_call(q, k, v, o, is_causal, sm_scale, k_lens, q_lens)
    nbytes = (C.c_uint64 * 2)()
    rc = lib.ksana_sage_train_attn_scratch(call, C.addressof(nbytes), C.addressof(nbytes) + 8)
    if rc != _capi.OK:
        _capi.check(rc, "train_ops.attention")
    with _on(q.device):
        scratch = _scratch(nbytes[0], q.device)
        rc = lib.ksana_sage_train_attn_fwd(call, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), _ptr(scratch), _stream_ptr(q.device))
    if rc != _capi.OK:
        _capi.check(rc, "train_ops.attention")
    return o, lse, nbytes[1]


def _attention_backward(do, q, k, v, o, lse, scratch_bytes, k_shape, is_causal, sm_scale, k_lens, q_lens, want_q: bool, want_kv: bool):
    dq = _contiguous_like(q) if want_q else None
    dk, dv = (_contiguous_like(k), _contiguous_like(k)) if want_kv else (None, None)
    if q.numel() == 0 or k.numel() == 0:
        return tuple(None if t is None else t.zero_() for t in (dq, dk, dv))
    shape, dtype, device = do.shape, do.dtype, do.get_device()
    if not (q.shape == shape and o.shape == shape and k.shape == k_shape and v.shape == k_shape
            and q.dtype is dtype and k.dtype is dtype and v.dtype is dtype and o.dtype is dtype
            and q.get_device() == device and k.get_device() == device and v.get_device() == device and o.get_device() == device):
        raise RuntimeError("a saved tensor came back from its hooks with another shape, type or device")
    # (the saved tensors too: see _kept)
    do, q, k, v, o = _readable(do), _readable(q), _readable(k), _readable(v), _readable(o)
    lse = _kept(lse, torch.float32, (shape[0], shape[2], shape[1]), device)
    k_lens, q_lens = _kept(k_lens, torch.int32, shape[:1], device), _kept(q_lens, torch.int32, shape[:1], device)
    call = _attention_call(q, k, v, o, is_causal, sm_scale, k_lens, q_lens)
    with _on(q.device):
        scratch = _scratch(scratch_bytes, q.device)
        rc = _capi.load().ksana_sage_train_attn_bwd(call, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), do.data_ptr(),
                                                    _STRIDES.pack(*do.stride()), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(scratch), _stream_ptr(q.device))
    if rc != _capi.OK:
        _capi.check(rc, "train_ops.attention, backward")
    return dq, dk, dv


class _Once(torch.autograd.Function):
    """Gradients on their way out of a backward pass that is itself recorded, and what they were formed from: differentiating them is refused.
    (torch's once_differentiable cuts them off from what they depend on: ``torch.autograd.functional.jvp`` then gives zeros.)"""

    @staticmethod
    def forward(ctx, number: int, *tensors):
        return tuple(t.view_as(t) for t in tensors[:number])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("train_ops: gradients of gradients are not available")


def _not_twice(grads: tuple, *sources: torch.Tensor | None) -> tuple:
    given = [t for t in grads if t is not None]
    if not given:
        return grads
    out = iter(_Once.apply(len(given), *given, *(t for t in sources if t is not None)))
    return tuple(None if t is None else next(out) for t in grads)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, is_causal, sm_scale, k_lens, q_lens):
        o, lse, scratch_bytes = _attention_forward(q, k, v, is_causal, sm_scale, k_lens, q_lens, True)
        ctx.save_for_backward(q, k, v, o, lse, k_lens, q_lens)
        ctx.options = (scratch_bytes, k.shape, is_causal, sm_scale)
        return o

    @staticmethod
    def backward(ctx, do):
        _refuse_unseen("attention's backward pass", do)
        if torch.is_grad_enabled():
            with torch.no_grad():
                d = _Attention.gradients(ctx, do)
            return _not_twice(d, do, *ctx.saved_tensors[:3])
        return _Attention.gradients(ctx, do)

    @staticmethod
    def gradients(ctx, do):
        want_q, want_k, want_v = ctx.needs_input_grad[:3]
        q, k, v, o, lse, k_lens, q_lens = ctx.saved_tensors
        dq, dk, dv = _attention_backward(do, q, k, v, o, lse, *ctx.options, k_lens, q_lens, want_q, want_k or want_v)
        return dq, dk if want_k else None, dv if want_v else None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tensor_layout: str = "NHD", is_causal: bool = False,
              sm_scale: float | None = None, k_lens=None, q_lens=None) -> torch.Tensor:
    """softmax(sm_scale q k^T) v with gradients for q, k and v: ``[B, L, H, D]`` ("NHD") or ``[B, H, L, D]`` ("HND") in and out,
    bf16 or fp16, head size 64 or 128, heads of q a multiple of those of k and v.

    ``k_lens``, ``q_lens``, ``is_causal`` and ``sm_scale`` mean what they mean for ``sageattn``; rows that see no key are zeros
    and give no gradient; keys and values behind ``k_lens[b]``, query rows and their gradients behind ``q_lens[b]`` are not
    read.  Int32 counts on the device are read by the kernels, in the backward pass again (writing to them in between is an
    error, as for the tensors).  Scores, softmax statistics and sums are fp32; probabilities and their gradients are rounded to the tensors' type
    where they are multiplied on, in fp16 scaled by powers of two that keep small gradients representable.  Keys that only causal masking
    hides have the weight 0, as in a product of matrices: not-a-numbers and infinities among them may show in the rows before."""
    if tensor_layout not in ("NHD", "HND"):
        raise ValueError(f"tensor_layout {tensor_layout!r} unknown")
    if tensor_layout == "HND":
        q, k, v = (t.transpose(1, 2) if t.dim() == 4 else t for t in (q, k, v))
    _check_attention(q, k, v)
    _refuse_unseen("attention", q, k, v)
    if sm_scale is not None and not abs(sm_scale) <= 2e38:
        raise ValueError(f"sm_scale {sm_scale} is not a number of at most 2e38 in size")
    k_lens, q_lens = (_k_lens_arg(n, q.shape[0], q.device, name) for n, name in ((k_lens, "k_lens"), (q_lens, "q_lens")))
    q, k, v = _readable(q), _readable(k), _readable(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o = _Attention.apply(q, k, v, bool(is_causal), sm_scale, k_lens, q_lens)
    else:
        o = _attention_forward(q, k, v, bool(is_causal), sm_scale, k_lens, q_lens, False)[0]
    return o.transpose(1, 2) if tensor_layout == "HND" else o


_NORMS = {None: _capi.NORM_NONE, "layer": _capi.NORM_LAYER, "rms": _capi.NORM_RMS}
_NORM_DTYPES = {torch.bfloat16: _capi.BF16, torch.float16: _capi.FP16, torch.float32: _capi.FP32}
_VECTORS = ("gate", "scale", "shift", "weight", "bias", "post_weight")  # in the order of the library's structure


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``[B, L, C]`` with contiguous channels and strides the kernels take (an expanded tensor has a stride of 0, which they do)."""
    return t if t.is_contiguous() or t.stride(2) == 1 and t.stride(0) >= 0 and t.stride(1) >= 0 else t.contiguous()


def _norm_call(x, y, vectors, norm, post_norm, residual_scale, eps, n_dtype) -> bytes:
    B, L, C_ = x.shape
    args = []
    for t in vectors:
        if t is None:
            args += (0, 0, 0, 0)
        else:
            args += (t.data_ptr(), t.stride(0) if t.dim() > 1 and t.shape[0] > 1 else 0, _NORM_DTYPES[t.dtype], 0)
    return _NORM.pack(B, L, C_, _NORM_DTYPES[x.dtype], _NORM_DTYPES[n_dtype], _NORMS[norm], _NORMS[post_norm], residual_scale, eps, 0,
                      *x.stride()[:2], *((0, 0) if y is None else y.stride()[:2]), *args)


def _residual_norm_forward(x, y, call, n_dtype, want_stats: bool):
    h = None if y is None else _contiguous_like(x)
    n = _contiguous_like(x) if n_dtype == x.dtype else torch.empty(x.shape, dtype=n_dtype, device=x.device)
    stats = torch.empty((*x.shape[:2], 4), dtype=torch.float32, device=x.device) if want_stats else None
    if x.numel() == 0:
        return h, n, stats
    with _on(x.device):
        rc = _capi.load().ksana_sage_train_norm_fwd(call, x.data_ptr(), _ptr(y), _ptr(h), n.data_ptr(), _ptr(stats), _stream_ptr(x.device))
    if rc != _capi.OK:
        _capi.check(rc, "train_ops.residual_norm")
    return h, n, stats


def _residual_norm_backward(ctx, grads) -> tuple:
    x, y, stats, *vectors = ctx.saved_tensors
    dh, dn = grads if y is not None else (None, grads[0])
    if dh is None and dn is None:
        return (None,) * 13
    options, like = ctx.options, dn if dh is None else dh
    n_dtype, shape, device = options[-1], like.shape, like.get_device()
    # (hooks may have laid the saved tensors out anew: see _kept.  All copies are held until the launches are made.)
    if x.shape != shape or x.get_device() != device or (dh is not None and x.dtype is not dh.dtype) or (
            y is not None and (y.shape != shape or y.dtype is not n_dtype or y.get_device() != device)):
        raise RuntimeError("a saved tensor came back from its hooks with another shape, type or device")
    x, y = _rows(x), None if y is None else _rows(y)
    vectors = [t if t is None or (t.is_contiguous() and t.shape == s and t.get_device() == device) else _norm_vector(name, t, x)
               for name, t, s in zip(_VECTORS, vectors, ctx.shapes)]
    stats = _kept(stats, torch.float32, (shape[0], shape[1], 4), device)
    call = _norm_call(x, y, vectors, *options)
    dn = torch.zeros(x.shape, dtype=n_dtype, device=x.device) if dn is None else dn.contiguous()
    dh = None if dh is None else dh.contiguous()
    dx, dy = _contiguous_like(x), None if y is None else _contiguous_like(y)
    d_vectors = [_contiguous_like(t) if t is not None and want else None for t, want in zip(vectors, ctx.needs_input_grad[2:8])]
    if x.numel() == 0:
        return (dx, dy, *(None if t is None else t.zero_() for t in d_vectors), *(None,) * 5)
    lib = _capi.load()
    nbytes, pointers = C.c_uint64(0), _POINTERS.pack(*[0 if t is None else t.data_ptr() for t in d_vectors])
    rc = lib.ksana_sage_train_norm_scratch(call, C.addressof(nbytes))
    if rc == _capi.OK:
        with _on(x.device):
            scratch = _scratch(nbytes.value, x.device)
            rc = lib.ksana_sage_train_norm_bwd(call, x.data_ptr(), _ptr(y), stats.data_ptr(), _ptr(dh), dn.data_ptr(), dx.data_ptr(), _ptr(dy),
                                               pointers, _ptr(scratch), _stream_ptr(x.device))
    if rc != _capi.OK:
        _capi.check(rc, "train_ops.residual_norm, backward")
    return (dx, dy, *d_vectors, *(None,) * 5)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, shift, weight, bias, post_weight, norm, post_norm, residual_scale, eps, n_dtype):
        vectors = (gate, scale, shift, weight, bias, post_weight)
        h, n, stats = _residual_norm_forward(x, y, _norm_call(x, y, vectors, norm, post_norm, residual_scale, eps, n_dtype), n_dtype, True)
        ctx.save_for_backward(x, y, stats, *vectors)
        ctx.options = (norm, post_norm, residual_scale, eps, n_dtype)
        ctx.shapes = [None if t is None else t.shape for t in vectors]
        ctx.set_materialize_grads(False)
        return n if y is None else (h, n)

    @staticmethod
    def backward(ctx, *grads):
        _refuse_unseen("residual_norm's backward pass", *grads)
        if torch.is_grad_enabled():
            with torch.no_grad():
                d = _residual_norm_backward(ctx, grads)
            x, y, _, *vectors = ctx.saved_tensors
            return _not_twice(d, *grads, x, y, *vectors)
        return _residual_norm_backward(ctx, grads)


def _wants_gradient(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _norm_vector(name: str, t: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor | None:
    """A vector as the kernels read it, its channels contiguous: ``[C]``, or ``[B, C]`` / ``[B, 1, C]`` with one for every batch entry or
    one for all of them (also slices of such a tensor, whose entries lie further apart)."""
    if t is None:
        return None
    B, _, C_ = x.shape
    if t.get_device() != x.get_device() or t.dtype not in _NORM_DTYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16 on {x.device}, got {t.dtype} on {t.device}")
    shape = t.shape
    if shape != (C_,):
        own = name in ("gate", "scale", "shift")
        if not (own and shape in ((B, C_), (1, C_), (B, 1, C_), (1, 1, C_))):
            raise ValueError(f"{name} must be [{C_}]" + (f", [{B}, {C_}] or [{B}, 1, {C_}]" if own else "") + f", got {tuple(shape)}")
    return t if t.is_contiguous() else _vector_rows(t)


def _vector_rows(t: torch.Tensor) -> torch.Tensor:
    """Contiguous channels; entries of their own any positive stride apart."""
    if t.stride(-1) != 1 and t.shape[-1] > 1 or t.dim() > 1 and t.shape[0] > 1 and t.stride(0) <= 0:
        return t.contiguous()
    return t


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, gate=None, residual_scale: float = 1.0, post_norm: str | None = None,
                  post_weight=None, norm: str = "layer", weight=None, bias=None, scale=None, shift=None, eps: float = 1e-6,
                  out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """What stands between two parts of a block, with gradients for every tensor: ``(h, n)`` with

    ``u = post_norm(y) * post_weight``, ``h = residual_scale * x + gate * u``, ``n = (norm(h) * weight + bias) * (1 + scale) + shift``

    for the residual stream ``x`` and the part's output ``y``, both ``[B, L, C]``; h goes on as the residual stream (x's type), n into the next
    part (y's type).  ``norm`` ("layer" or "rms") and ``post_norm`` (None, "layer" or "rms") run over the channels, ``eps`` under both
    roots.  ``gate``, ``scale`` and ``shift`` are ``[C]``, ``[B, C]`` or ``[B, 1, C]``; ``weight``, ``bias`` and ``post_weight`` ``[C]``; any of
    them absent, each in fp32, fp16 or bf16.  Without ``y``, at a block's first part, h is x itself and n of ``out_dtype`` (x's type by
    default, or a half type under an fp32 stream).  x and y share a type, or x is fp32.  At most 8192 channels.

    Statistics and arithmetic are fp32, n comes from the unrounded h, and every result and gradient is rounded once."""
    if x.dim() != 3 or (y is not None and y.shape != x.shape):
        raise ValueError(f"residual_norm expects x and y of one shape [B, L, C], got {tuple(x.shape)}" + ("" if y is None else f" and {tuple(y.shape)}"))
    if norm not in ("layer", "rms") or post_norm not in _NORMS:
        raise ValueError(f"norm {norm!r} / post_norm {post_norm!r} unknown")
    for t in (x,) if y is None else (x, y):
        if not t.is_cuda:
            raise RuntimeError(f"residual_norm needs tensors on a HIP device; there is no CPU path (got device {t.device})")
        if t.dtype not in _NORM_DTYPES or t.get_device() != x.get_device():
            raise ValueError(f"x and y must be float32, float16 or bfloat16 on one device, got {t.dtype} on {t.device}")
    if y is None:
        if gate is not None or post_norm is not None or post_weight is not None or residual_scale != 1.0:
            raise ValueError("gate, post_norm, post_weight and residual_scale go with y")
        n_dtype = x.dtype if out_dtype is None else out_dtype
    else:
        n_dtype = y.dtype
        if out_dtype not in (None, n_dtype):
            raise ValueError(f"with y the normalised result has its type, {n_dtype}")
    if n_dtype not in _NORM_DTYPES or n_dtype != x.dtype and x.dtype != torch.float32:
        raise ValueError(f"x of {x.dtype} does not go with {n_dtype}")
    if post_weight is not None and post_norm is None:
        raise ValueError("post_weight goes with post_norm")
    if x.shape[2] == 0:
        raise ValueError("residual_norm needs at least one channel")
    _refuse_unseen("residual_norm", x, y, gate, scale, shift, weight, bias, post_weight)
    vectors = [_norm_vector(name, t, x) for name, t in zip(_VECTORS, (gate, scale, shift, weight, bias, post_weight))]
    x_rows, y_rows = _rows(x), None if y is None else _rows(y)
    residual_scale, eps = float(residual_scale), float(eps)
    if torch.is_grad_enabled() and _wants_gradient(x, y, *vectors):
        out = _ResidualNorm.apply(x_rows, y_rows, *vectors, norm, post_norm, residual_scale, eps, n_dtype)
        return (x, out) if y is None else out
    call = _norm_call(x_rows, y_rows, vectors, norm, post_norm, residual_scale, eps, n_dtype)
    h, n, _ = _residual_norm_forward(x_rows, y_rows, call, n_dtype, False)
    return (x if y is None else h), n


# ------------------------------------------------------------------------------------------------ rotary positions

_ROTARY = struct.Struct("=15if15q2Q")  # ksana_sage_rotary
_MOST_AXES = 4


def rotary_frequencies(width: int, base: float = 10000.0, *, sections=None, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, low: float = 1.0, high: float = 32.0, device="cuda") -> torch.Tensor:
    """The radians that each of ``width // 2`` pairs turns by from one position to the next, float64 as ``rotary`` takes them:
    ``base ** (-i / n)`` for pair i of n; with ``sections`` the n pairs of every axis by themselves.

    For sequences ``factor`` times as long as a model was trained on, ``scaling`` is "linear" (all frequencies divided by the factor), "base" (the
    base raised so that the slowest pair's is divided by it) or "parts" (pairs that make ``high`` turns and more over ``original_length`` positions
    keep theirs, those that make ``low`` and fewer have it divided, between them it goes over evenly with the number of turns)."""
    sections = (width // 2,) if sections is None else tuple(sections)
    if width < 2 or width % 2 or sum(sections) != width // 2 or min(sections) < 0:
        raise ValueError(f"width {width} is not even, or its pairs are not those of sections {sections}")
    if scaling not in (None, "linear", "base", "parts") or not factor > 0.0:
        raise ValueError(f"scaling {scaling!r} with factor {factor} unknown")
    parts = []
    for n in sections:
        i = torch.arange(n, dtype=torch.float64) / max(n, 1)
        own = base * factor ** (n / (n - 1)) if scaling == "base" and n > 1 else base
        parts.append(torch.pow(torch.tensor(own, dtype=torch.float64), -i))
    f = torch.cat(parts)
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if original_length is None or not 0.0 < low < high:
            raise ValueError("scaling by parts goes with original_length and 0 < low < high")
        kept = ((f * (original_length / (2.0 * torch.pi)) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * kept + f / factor * (1.0 - kept)
    return f.to(device)


def _channels_last(t: torch.Tensor) -> torch.Tensor:
    """``[B, L, H, D]`` with contiguous channels and strides that are not negative."""
    return t if t.is_contiguous() or t.stride(3) == 1 and min(t.stride()[:3]) >= 0 else t.contiguous()


def _check_rotary(frequencies, positions, sections, B: int, L: int, D: int, device: int) -> tuple:
    """(axes, ends of the axes' pairs, whether positions have an axis behind) as the library takes them."""
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or frequencies.get_device() != device or not frequencies.is_contiguous():
        raise ValueError(f"frequencies must be a contiguous vector of float64 on the tensors' device, got {frequencies.dtype} {tuple(frequencies.shape)} on {frequencies.device}")
    if frequencies.requires_grad:
        raise ValueError("frequencies have no gradient here")
    pairs = frequencies.shape[0]
    if not 1 <= pairs <= D // 2:
        raise ValueError(f"{pairs} frequencies do not go with heads of {D} channels")
    axes, ends, end = 1 if sections is None else len(sections), [], 0
    for n in (pairs,) if sections is None else sections:
        if n < 0:
            raise ValueError(f"sections {sections} hold a negative number")
        end += n
        ends.append(end)
    if not 1 <= axes <= _MOST_AXES or end != pairs:
        raise ValueError(f"sections {sections} must be at most {_MOST_AXES} numbers of pairs, {pairs} in all")
    if positions is not None:
        lead = () if sections is None else (axes,)
        if positions.dtype not in (torch.int32, torch.int64) or positions.get_device() != device or positions.shape not in ((L, *lead), (1, L, *lead), (B, L, *lead)):
            raise ValueError(f"positions must be int32 or int64 [{L}] or [{B}, {L}]{f' with {axes} axes behind' if lead else ''} on the tensors' device, "
                             f"got {positions.dtype} {tuple(positions.shape)} on {positions.device}")
    return axes, ends + [0] * (_MOST_AXES - axes), sections is not None


def _position_strides(positions: torch.Tensor | None, with_axes: bool) -> tuple:
    if positions is None:
        return 0, 0, 0
    strides = positions.stride() if with_axes else (*positions.stride(), 0)
    return (0, *strides) if len(strides) == 2 else (strides[0] if positions.shape[0] > 1 else 0, *strides[1:])


_NO_ROWS = (0, 0, 0, 1)


def _rotary_call(q, k, v, frequencies, positions, checked, interleaved: bool, magnitude: float, inverse: bool) -> bytes:
    x = k if q is None else q
    B, L, _, D = x.shape
    axes, ends, with_axes = checked
    return _ROTARY.pack(B, L, D, 0 if q is None else q.shape[2], 0 if k is None else k.shape[2], _NORM_DTYPES[x.dtype],
                        0 if frequencies is None else 2 * frequencies.shape[0], interleaved, inverse, axes, *ends,
                        positions is not None and positions.dtype is torch.int64, magnitude, *(_NO_ROWS if q is None else q.stride()),
                        *(_NO_ROWS if k is None else k.stride()), *(_NO_ROWS if v is None else v.stride()), *_position_strides(positions, with_axes),
                        0 if positions is None else positions.data_ptr(), 0 if frequencies is None else frequencies.data_ptr())


def _turn(q, k, frequencies, positions, checked, interleaved, magnitude, inverse) -> tuple:
    q_out, k_out = _contiguous_like(q), None if k is None else _contiguous_like(k)
    q_rows = None if q.numel() == 0 else _channels_last(q)
    k_rows = None if k is None or k.numel() == 0 else _channels_last(k)
    if q_rows is None and k_rows is None:
        return q_out, k_out
    call, device = _rotary_call(q_rows, k_rows, None, frequencies, positions, checked, interleaved, magnitude, inverse), q.device
    with _on(device):
        rc = _capi.load().ksana_sage_rotary_rows(call, _ptr(q_rows), _ptr(k_rows), q_out.data_ptr(), _ptr(k_out), _stream_ptr(device))
    if rc != _capi.OK:
        _capi.check(rc, "train_ops.rotary")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """Its gradients are turned back by the function itself, so that they have gradients too."""

    @staticmethod
    def forward(ctx, q, k, frequencies, positions, checked, interleaved, magnitude, inverse):
        ctx.save_for_backward(frequencies, positions)
        ctx.options = (checked, interleaved, magnitude, inverse)
        ctx.was = (frequencies.shape, None if positions is None else (positions.dtype, positions.shape))
        ctx.set_materialize_grads(False)
        q, k = _turn(q, k, frequencies, positions, *ctx.options)
        return q if k is None else (q, k)

    @staticmethod
    def backward(ctx, dq, dk=None):
        _refuse_unseen("rotary's backward pass", dq, dk)
        want_q, want_k = ctx.needs_input_grad[:2]
        given = [t for t, want in ((dq, want_q), (dk, want_k)) if want and t is not None]
        if not given:
            return (None,) * 8
        frequencies, positions = ctx.saved_tensors
        device = given[0].get_device()
        frequencies = _kept(frequencies, torch.float64, ctx.was[0], device)
        if positions is not None:
            positions = _kept(positions, *ctx.was[1], device)
        checked, interleaved, magnitude, inverse = ctx.options
        turn = _Rotary.apply if torch.is_grad_enabled() else _turn
        out = turn(given[0], given[1] if len(given) > 1 else None, frequencies, positions, checked, interleaved, magnitude, not inverse)
        out = iter(out if isinstance(out, tuple) else (out,))
        return (next(out) if want_q and dq is not None else None, next(out) if want_k and dk is not None else None, *(None,) * 6)


def rotary(q: torch.Tensor, k: torch.Tensor | None = None, *, frequencies: torch.Tensor, positions: torch.Tensor | None = None, sections=None,
           interleaved: bool = True, magnitude: float = 1.0, tensor_layout: str = "NHD") -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions of ``q`` - and of ``k``, in the same pass - with gradients: ``[B, L, H, D]`` ("NHD") or ``[B, H, L, D]`` ("HND") in and out, bf16, fp16 or
    fp32, any strides, heads of up to 512 channels.

    Of every head the first ``2 * len(frequencies)`` channels turn, in pairs: channels 2 i and 2 i + 1 (``interleaved``) or i and i + len(frequencies);
    the others are copied.  Pair i of a token turns by its position times ``frequencies[i]`` radians (float64, see ``rotary_frequencies``), and
    ``magnitude`` is multiplied on.  ``positions``: int32 or int64, ``[L]`` or ``[B, L]``, negative ones too; 0, 1, .. by default.  With ``sections``,
    as (22, 21, 21) for a video's frames, rows and columns, the first 22 pairs go by the first of a token's positions, ``[L, 3]`` or ``[B, L, 3]``,
    and so on.

    Angles are formed in 64 bits, everything else in fp32, and results and gradients are rounded once: cosines and sines are off by a few 2^-24, and by about 2^-52 of the
    angle, position times frequency, which is less up to 2^28 radians (2e-4 at 10^12, and of no use at 10^15)."""
    if tensor_layout not in ("NHD", "HND"):
        raise ValueError(f"tensor_layout {tensor_layout!r} unknown")
    for t in (q,) if k is None else (q, k):
        if t.dim() != 4:
            raise ValueError("rotary expects 4-D tensors")
        if not t.is_cuda:
            raise RuntimeError(f"rotary needs tensors on a HIP device; there is no CPU path (got device {t.device})")
        if t.dtype not in _NORM_DTYPES or t.dtype != q.dtype or t.get_device() != q.get_device():
            raise ValueError(f"q and k must be float32, float16 or bfloat16 of one type on one device, got {t.dtype} on {t.device}")
    if tensor_layout == "HND":
        q, k = q.transpose(1, 2), None if k is None else k.transpose(1, 2)
    B, L, _, D = q.shape
    if k is not None and (k.shape[:2] != q.shape[:2] or k.shape[3] != D):
        raise ValueError(f"incompatible shapes q{tuple(q.shape)} k{tuple(k.shape)}")
    checked, magnitude = _check_rotary(frequencies, positions, sections, B, L, D, q.get_device()), float(magnitude)
    if not abs(magnitude) <= 3e38:
        raise ValueError(f"magnitude {magnitude} is not a number of fp32")
    _refuse_unseen("rotary", q, k)
    if torch.is_grad_enabled() and _wants_gradient(q, k):
        out = _Rotary.apply(q, k, frequencies, positions, checked, bool(interleaved), magnitude, False)
    else:
        out = _turn(q, k, frequencies, positions, checked, bool(interleaved), magnitude, False)
        out = out[0] if k is None else out
    if tensor_layout == "HND":
        return out.transpose(1, 2) if k is None else (out[0].transpose(1, 2), out[1].transpose(1, 2))
    return out
