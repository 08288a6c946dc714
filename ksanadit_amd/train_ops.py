"""Operators with gradients: what a block's attention half needs where it is trained, next to ``sage_ops`` that generates.

``attention`` takes the place of ``sageattn`` where gradients are wanted: the same layouts, key and query counts and causal
masking, 16-bit products without quantization, and a backward pass that recomputes the probabilities.
``residual_norm`` is what stands between two parts of a block: gate, residual sum, norm and modulation in one pass.

Both run on the tensors' HIP device, on torch's current stream there, without synchronising; scratch comes from torch's caching
allocator.  Repeated calls give the same bits.  Gradients of gradients are refused.
"""

from __future__ import annotations

import ctypes as C
from contextlib import nullcontext

import torch
from torch.autograd.function import once_differentiable

from . import _capi
from .sage_ops import _DTYPES, _k_lens_arg, _require_hip, _stream_ptr, _strides, _usable


def _on(device: torch.device):
    """The device made current where it is not: kernels start on the current one."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _scratch(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


class _AttentionCall:
    """The library's structure for tensors ``[B, L, H, D]`` as the kernels read them, and its scratch sizes."""

    __slots__ = ("c", "lens", "fwd_bytes", "bwd_bytes")

    def __init__(self, q, k, v, o, is_causal: bool, sm_scale: float | None, k_lens, q_lens):
        B, Lq, Hq, D = q.shape
        self.lens = (k_lens, q_lens)  # (alive as long as the structure points to them)
        self.c = _capi.TrainAttn(_capi.Shape(B, Hq, k.shape[2], Lq, k.shape[1], D), _DTYPES[q.dtype], int(is_causal),
                                 D**-0.5 if sm_scale is None else float(sm_scale), 0, _strides(q), _strides(k), _strides(v), _strides(o),
                                 _ptr(q_lens), _ptr(k_lens))
        fwd, bwd = C.c_uint64(0), C.c_uint64(0)
        _capi.check(_capi.load().ksana_sage_train_attn_scratch(C.addressof(self.c), C.addressof(fwd), C.addressof(bwd)), "train_ops.attention")
        self.fwd_bytes, self.bwd_bytes = fwd.value, bwd.value


def _check_attention(q, k, v) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention expects 4-D tensors")
    _require_hip(q, k, v)
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"incompatible shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")


def _attention_forward(q, k, v, is_causal, sm_scale, k_lens, q_lens, want_lse: bool):
    """(o, lse or None, the call) of ``[B, L, H, D]`` tensors the kernels can read."""
    B, Lq, Hq, D = q.shape
    o = torch.empty((B, Lq, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=q.device) if want_lse else None
    if q.numel() == 0 or k.numel() == 0:
        return o.zero_(), None if lse is None else lse.fill_(-torch.inf), None
    call = _AttentionCall(q, k, v, o, is_causal, sm_scale, k_lens, q_lens)
    with _on(q.device):
        scratch = _scratch(call.fwd_bytes, q.device)
        rc = _capi.load().ksana_sage_train_attn_fwd(C.addressof(call.c), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse),
                                                    _ptr(scratch), _stream_ptr(q.device))
    _capi.check(rc, "train_ops.attention")
    return o, lse, call


def _attention_backward(do, q, k, v, o, lse, call, want_q: bool, want_kv: bool):
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if want else None
                  for t, want in ((q, want_q), (k, want_kv), (v, want_kv)))
    if q.numel() == 0 or k.numel() == 0:
        return tuple(None if t is None else t.zero_() for t in (dq, dk, dv))
    do = _usable(do)
    with _on(q.device):
        scratch = _scratch(call.bwd_bytes, q.device)
        rc = _capi.load().ksana_sage_train_attn_bwd(C.addressof(call.c), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(),
                                                    do.data_ptr(), _strides(do), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(scratch), _stream_ptr(q.device))
    _capi.check(rc, "train_ops.attention, backward")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, is_causal, sm_scale, k_lens, q_lens):
        o, lse, call = _attention_forward(q, k, v, is_causal, sm_scale, k_lens, q_lens, True)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.call = call
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        want_q, want_k, want_v = ctx.needs_input_grad[:3]
        dq, dk, dv = _attention_backward(do, *ctx.saved_tensors, ctx.call, want_q, want_k or want_v)
        return dq, dk if want_k else None, dv if want_v else None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tensor_layout: str = "NHD", is_causal: bool = False,
              sm_scale: float | None = None, k_lens=None, q_lens=None) -> torch.Tensor:
    """softmax(sm_scale q k^T) v with gradients for q, k and v: ``[B, L, H, D]`` ("NHD") or ``[B, H, L, D]`` ("HND") in and out,
    bf16 or fp16, head size 64 or 128, heads of q a multiple of those of k and v.

    ``k_lens``, ``q_lens``, ``is_causal`` and ``sm_scale`` mean what they mean for ``sageattn``; rows that see no key are zeros
    and give no gradient; keys and values behind ``k_lens[b]``, query rows and their gradients behind ``q_lens[b]`` are not
    read.  Counts on the device are taken as they are when the kernels run, also in the backward pass: they must not be
    written between the two.  Scores, softmax statistics and sums are fp32; probabilities and their gradients are rounded to the tensors' type
    where they are multiplied on, in fp16 scaled by powers of two that keep small gradients representable."""
    if tensor_layout not in ("NHD", "HND"):
        raise ValueError(f"tensor_layout {tensor_layout!r} unknown")
    if tensor_layout == "HND":
        q, k, v = (t.transpose(1, 2) if t.dim() == 4 else t for t in (q, k, v))
    _check_attention(q, k, v)
    k_lens, q_lens = (_k_lens_arg(n, q.shape[0], q.device, name) for n, name in ((k_lens, "k_lens"), (q_lens, "q_lens")))
    q, k, v = _usable(q), _usable(k), _usable(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o = _Attention.apply(q, k, v, bool(is_causal), sm_scale, k_lens, q_lens)
    else:
        o = _attention_forward(q, k, v, bool(is_causal), sm_scale, k_lens, q_lens, False)[0]
    return o.transpose(1, 2) if tensor_layout == "HND" else o
