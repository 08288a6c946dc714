"""A paged cache of keys and values, for blocks that generate chunk by chunk: frames of a video, tokens of a text.

``append`` stores the keys and values of a chunk, and gives them and q their rotary positions on the way; ``attention`` is that of the chunk's queries on
everything their sequences have in the cache.  Both take the same table and counts:

    k_lens[b]  tokens of sequence b with the chunk's,   q_lens[b]  those of the chunk (all rows of q by default),
    pages[b]   the pages that hold the sequence's tokens, in order: token t is in page ``pages[b, t // page_size]``, slot ``t % page_size``

so row i of the chunk stands at position ``k_lens[b] - q_lens[b] + i``.  Every layer has a cache of its own; table and counts are the same for all of them.

Both run on the tensors' HIP device, on torch's current stream there; scratch comes from torch's caching allocator.  They do not synchronise and may be captured into a
graph, with counts as int32 tensors on that device (others are copied there in the call, which waits for the copy and cannot be captured); table and counts are read by the
kernels, so that replays go by what they hold then.  Counts below 0 are 0, and ``q_lens`` are at most the call's rows.  ``k_lens`` beyond ``entries * page_size``, more tokens than
the table has room for, are the caller's error, which calls that do not synchronise cannot report.  Both stay within the table then, but do not agree: ``append`` turns and stores rows by
their positions and leaves out those behind the table's end, ``attention`` takes that end as the sequence's.  Repeated calls give the same
bits.  There is no backward pass: ``train_ops`` has those.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch
from torch.autograd.graph import increment_version

from . import _capi
from .sage_ops import _DTYPES, _k_lens_arg, _stream_ptr
from .train_ops import _channels_last, _check_rotary, _contiguous_like, _on, _ptr, _readable, _refuse_unseen, _rotary_call, _scratch

# The library's structures, packed (see train_ops)
_CACHE = struct.Struct("=4Q3q4iQq2Q")  # ksana_sage_cache
_ATTENTION = struct.Struct("=7if8q")  # ksana_sage_cache_attn


class PagedCache(NamedTuple):
    """One layer's keys and values: ``[pages, heads, page_size, head_size]``, of the tensors' type (bf16, fp16) or float8_e4m3fn, head size 64 or 128; pages, heads and
    slots may lie any multiple of 16 bytes apart, the same in both.  ``k_scale`` and ``v_scale``, float32 ``[heads]``, positive: what an 8-bit cache's
    number 1 stands for (1 without)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None


def allocate(pages: int, page_size: int, heads: int, head_size: int, dtype: torch.dtype = torch.bfloat16, device="cuda", k_scale=None, v_scale=None) -> PagedCache:
    """A cache of ``pages`` pages, its contents as they come: nothing is read that was not stored."""
    shape = (pages, heads, page_size, head_size)
    return PagedCache(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device), k_scale, v_scale)


def _check_cache(cache: PagedCache, pages: torch.Tensor, x: torch.Tensor, heads: int | None) -> int:
    """The cache's type as the library takes it; x: rows of q or k."""
    k, v, k_scale, v_scale = cache
    device, dtype, shape = x.get_device(), k.dtype, k.shape
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype or k.stride() != v.stride() or k.get_device() != device or v.get_device() != device:
        raise ValueError(f"the cache must be two tensors [pages, heads, page_size, head_size] laid out alike on {x.device}, "
                         f"got {k.dtype} {tuple(k.shape)} on {k.device} and {v.dtype} {tuple(v.shape)} on {v.device}")
    if dtype != x.dtype and dtype != torch.float8_e4m3fn:
        raise ValueError(f"a cache of {dtype} does not go with {x.dtype}")
    if shape[3] != x.shape[3] or (heads is not None and shape[1] != heads):
        raise ValueError(f"the cache holds {shape[1]} heads of {shape[3]} channels, the tensors {x.shape[2]} of {x.shape[3]}")
    if k.numel() == 0 or k.stride(3) != 1 or k.requires_grad or v.requires_grad:
        raise ValueError("the cache must not be empty nor require gradients, and its channels must be contiguous")
    if k_scale is not None or v_scale is not None:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None and (dtype != torch.float8_e4m3fn or t.dtype != torch.float32 or t.shape != shape[1:2] or t.get_device() != device or not t.is_contiguous()):
                raise ValueError(f"{name} must be contiguous float32 [{shape[1]}] on {x.device}, for a float8_e4m3fn cache")
    if pages.dtype != torch.int32 or pages.dim() != 2 or pages.shape[0] != x.shape[0] or pages.get_device() != device or pages.shape[1] == 0 or (
            pages.stride(1) != 1 and pages.shape[1] > 1):
        raise ValueError(f"pages must be int32 [{x.shape[0]}, entries] with contiguous entries on {x.device}, got {pages.dtype} {tuple(pages.shape)} on {pages.device}")
    return _capi.E4M3 if dtype == torch.float8_e4m3fn else _DTYPES[dtype]


def _cache_call(cache: PagedCache, kind: int, pages, q_lens, k_lens) -> bytes:
    k = cache.k
    shape, strides = k.shape, k.stride()
    return _CACHE.pack(k.data_ptr(), cache.v.data_ptr(), 0 if cache.k_scale is None else cache.k_scale.data_ptr(), 0 if cache.v_scale is None else cache.v_scale.data_ptr(),
                       strides[0], strides[1], strides[2], shape[0], shape[2], kind, pages.shape[1], pages.data_ptr(), pages.stride(0),
                       0 if q_lens is None else q_lens.data_ptr(), k_lens.data_ptr())


def _check_rows(name: str, *tensors: torch.Tensor) -> None:
    first, wanted = tensors[0], False
    dtype, device = first.dtype, first.get_device()
    for t in tensors:
        if t.dim() != 4:
            raise ValueError(f"{name} expects 4-D tensors")
        if not t.is_cuda:
            raise RuntimeError(f"{name} needs tensors on a HIP device; there is no CPU path (got device {t.device})")
        if t.dtype != dtype or dtype not in _DTYPES or t.get_device() != device:
            raise ValueError(f"{name} takes bfloat16 or float16 tensors of one type on one device, got {t.dtype} on {t.device}")
        wanted = wanted or t.requires_grad
    if wanted and torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad(), or train with train_ops")


def _counts(counts, name: str, batch: int, x: torch.Tensor) -> torch.Tensor | None:
    """Counts as the kernels read them; those that are so already cost nothing."""
    if isinstance(counts, torch.Tensor) and counts.dtype is torch.int32 and counts.shape == (batch,) and counts.get_device() == x.get_device() and counts.is_contiguous():
        return counts
    return _k_lens_arg(counts, batch, x.device, name)


def append(k: torch.Tensor, v: torch.Tensor, cache: PagedCache, pages: torch.Tensor, k_lens, q_lens=None, *, q: torch.Tensor | None = None,
           frequencies: torch.Tensor | None = None, positions: torch.Tensor | None = None, sections=None, interleaved: bool = True,
           magnitude: float = 1.0) -> torch.Tensor | None:
    """Stores a chunk's ``k`` and ``v``, ``[B, L, heads, D]``, in the cache, row i of sequence b at position ``k_lens[b] - q_lens[b] + i``, and returns ``q``
    (``[B, L, Hq, D]``) with its rotary positions, or None without q.

    ``frequencies``, ``sections``, ``interleaved`` and ``magnitude`` are those of ``train_ops.rotary`` and turn k and q; so do ``positions``, which are by
    default the rows' own in their sequences.  Without ``frequencies`` nothing turns, and q is not taken.  An 8-bit cache gets the
    nearest of its numbers to the value (a key as it is turned, in fp32) divided by the scale, beyond the largest that one.

    Rows behind ``q_lens[b]`` are not stored, and zeros in the result.  Nor are rows at negative positions, behind the table's end or in pages that do not exist
    (entries that are negative or not below the cache's pages).  A page that is written to belongs to one sequence and stands in its table once."""
    _check_rows("append", *((k, v) if q is None else (k, v, q)))
    B, L, H, D = k.shape
    if v.shape != k.shape or (q is not None and (q.shape[:2] != k.shape[:2] or q.shape[3] != D)):
        raise ValueError(f"incompatible shapes k{tuple(k.shape)} v{tuple(v.shape)}" + ("" if q is None else f" q{tuple(q.shape)}"))
    kind = _check_cache(cache, pages, k, H)
    if frequencies is None:
        if q is not None or positions is not None or sections is not None:
            raise ValueError("q, positions and sections go with frequencies")
        checked = (1, (0, 0, 0, 0), False)
    else:
        checked = _check_rotary(frequencies, positions, sections, B, L, D, k.get_device())
    if not abs(magnitude) <= 3e38:
        raise ValueError(f"magnitude {magnitude} is not a number of fp32")
    if k_lens is None:
        raise ValueError("k_lens is needed: how many tokens every sequence has")
    _refuse_unseen("append", k, v, q)
    k_lens, q_lens = _counts(k_lens, "k_lens", B, k), _counts(q_lens, "q_lens", B, k)
    out = None if q is None else _contiguous_like(q)
    if k.numel() == 0:
        return out if out is None or out.numel() == 0 else out.zero_()
    k, v = _channels_last(k), _channels_last(v)
    q = None if q is None or q.shape[2] == 0 else _channels_last(q)
    call = _rotary_call(q, k, v, frequencies, positions, checked, bool(interleaved), float(magnitude), False)
    with _on(k.device):
        rc = _capi.load().ksana_sage_cache_append(call, _cache_call(cache, kind, pages, q_lens, k_lens), _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(out), _stream_ptr(k.device))
    if rc != _capi.OK:
        _capi.check(rc, "cache_ops.append")
    if not cache.k.is_inference() and not cache.v.is_inference():
        increment_version((cache.k, cache.v))  # (autograd notices writes to what it has saved)
    return out


def attention(q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, k_lens, q_lens=None, *, is_causal: bool = True,
              sm_scale: float | None = None) -> torch.Tensor:
    """softmax(sm_scale q k^T) v of a chunk's queries ``[B, L, Hq, D]``, the last ``q_lens[b]`` tokens of every sequence, on its ``k_lens[b]`` keys in the
    cache; ``is_causal``: on those up to a query's own position.  Hq is a multiple of the cache's heads.

    ``sm_scale`` is ``D ** -0.5`` by default.  Rows behind ``q_lens[b]`` and rows that see no key are zeros.  Keys behind ``k_lens[b]`` are not read, and keys in pages that
    do not exist (entries that are negative or not below the cache's pages) are not seen.  Scores, softmax statistics and sums are fp32; probabilities are rounded to q's type
    where they are multiplied on (in two parts on 16-bit caches, up to 32 rows to a key head).  Over n keys fp32's sums are off by about 2^-29 n of
    themselves if all roundings go one way, half a step of fp16 at 2^18 keys; where they do not, by far less.  Keys that only causal masking hides have the weight 0, as in a product of matrices:
    not-a-numbers and infinities among them may show in the rows before."""
    _check_rows("attention", q)
    kind = _check_cache(cache, pages, q, None)
    B, L, H, D = q.shape
    if H % cache.k.shape[1]:
        raise ValueError(f"{H} query heads are no multiple of the cache's {cache.k.shape[1]}")
    if sm_scale is not None and not abs(sm_scale) <= 2e38:
        raise ValueError(f"sm_scale {sm_scale} is not a number of at most 2e38 in size")
    if k_lens is None:
        raise ValueError("k_lens is needed: how many tokens every sequence has")
    _refuse_unseen("attention", q)
    k_lens, q_lens = _counts(k_lens, "k_lens", B, q), _counts(q_lens, "q_lens", B, q)
    o = _contiguous_like(q)
    if q.numel() == 0:
        return o
    q = _readable(q)
    call = _ATTENTION.pack(B, H, cache.k.shape[1], L, D, _DTYPES[q.dtype], bool(is_causal), D**-0.5 if sm_scale is None else sm_scale, *q.stride(), *o.stride())
    held = _cache_call(cache, kind, pages, q_lens, k_lens)
    lib, nbytes = _capi.load(), C.c_uint64(0)
    rc = lib.ksana_sage_cache_attn_scratch(call, held, C.addressof(nbytes))
    if rc == _capi.OK:
        with _on(q.device):
            scratch = _scratch(nbytes.value, q.device)
            rc = lib.ksana_sage_cache_attn_fwd(call, held, q.data_ptr(), o.data_ptr(), _ptr(scratch), _stream_ptr(q.device))
    if rc != _capi.OK:
        _capi.check(rc, "cache_ops.attention")
    return o
