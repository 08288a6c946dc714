"""The attention operator the DiT blocks hold: ``op(q, k, v, **kwargs) -> o`` on ``[B, L, H, D]``.

Same contract as ksana/operations/attention/attention_op.py:24-91: the default softmax scale is
``head_size ** -0.5`` (:39), a missing config is a ``ValueError`` (:41-42), the backend object is
built lazily on the first call and rebuilt when the input dtype changes (:53-70), inputs that are
not 4-D are a ``ValueError`` (:80-81), backend kwargs pass through untouched (:86-91), and the
forward is kept out of Dynamo graphs (:72).

Beyond it: ``trainable=True`` asks for a backend with a backward pass.  The Sage backend then runs ``train_ops.attention`` where its inputs
require gradients, torch's SDPA has one as it is, and a backend without one is a ``ValueError``.
``op(q, k, v, kv_cache=.., pages=.., k_lens=..)`` attends through a paged cache (``cache_ops``) where the Sage backend runs; elsewhere it is a ``ValueError``.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from .backends import KsanaAttentionBackendImpl, get_attention_backend_impl
from .config import KsanaAttentionBackend, KsanaAttentionConfig
from .logger import log

_TRAINABLE = (KsanaAttentionBackend.SAGE_ATTN, KsanaAttentionBackend.TORCH_SDPA)
_CACHED = (KsanaAttentionBackend.SAGE_ATTN,)


class KsanaAttentionOp(nn.Module):
    def __init__(self, num_heads: int, head_size: int, *, num_kv_heads: int | None = None,
                 softmax_scale: float | None = None, causal: bool = False,
                 attention_config: KsanaAttentionConfig = None, trainable: bool = False) -> None:
        super().__init__()
        if attention_config is None:
            raise ValueError("attention_config should not be None")
        log.debug(f"KsanaAttentionOp with config: {attention_config}")
        self.attention_config = attention_config
        self.num_heads, self.head_size, self.causal = num_heads, head_size, causal
        self.num_kv_heads = num_heads if not num_kv_heads else num_kv_heads
        self.softmax_scale = head_size**-0.5 if softmax_scale is None else softmax_scale
        self.trainable = bool(trainable)
        # the backend object and the input dtype it was picked for
        self._attn_impl: KsanaAttentionBackendImpl | None = None
        self._attn_impl_dtype: torch.dtype | None = None

    @property
    def backend_type(self):
        impl = self._attn_impl
        return impl.type() if impl is not None else None

    def _ensure_impl(self, dtype: torch.dtype) -> None:
        """Pick and build the backend on first use, again when the input dtype changes (a backend may support one
        dtype and not another)."""
        if self._attn_impl is None or self._attn_impl_dtype != dtype:
            cls = get_attention_backend_impl(attention_config=self.attention_config, head_size=self.head_size,
                                             dtype=dtype)
            if self.trainable and cls.type() not in _TRAINABLE:
                raise ValueError(f"attention backend {cls.type()} has no backward pass (trainable=True)")
            self._attn_impl = cls(attention_config=self.attention_config, num_heads=self.num_heads,
                                  head_size=self.head_size, causal=self.causal, softmax_scale=self.softmax_scale,
                                  num_kv_heads=self.num_kv_heads, **({"trainable": True} if self.trainable else {}))
            self._attn_impl_dtype = dtype

    @torch.compiler.disable
    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, **backend_kwargs) -> torch.Tensor:
        if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
            raise ValueError("LocalAttentionOp expects tensors shaped [B, L, H, D].")
        self._ensure_impl(query.dtype)
        if backend_kwargs.get("kv_cache") is not None and self.backend_type not in _CACHED:
            raise ValueError(f"attention backend {self.backend_type} has no paged cache (kv_cache)")
        return self._attn_impl.forward(query, key, value, **backend_kwargs)
