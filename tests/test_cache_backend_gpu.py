"""Models of other types than the caches they attend through."""

import pytest
import torch

from ksanadit_amd import KsanaAttentionConfig, cache_ops, pick_attn_op, train_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("turned", [True, False])
def test_an_fp32_model_goes_by_its_cache(hip_device, kind, turned):
    """Bit for bit the calls on tensors of the cache's type, of bf16 on 8-bit ones; the result has the model's."""
    of = torch.float16 if kind == torch.float16 else torch.bfloat16
    q, k, v = (torch.randn(1, 20, h, 128, device=hip_device) for h in (4, 2, 2))
    pages, lens = torch.arange(2, dtype=torch.int32, device=hip_device)[None], torch.tensor([20], dtype=torch.int32, device=hip_device)
    f = {"frequencies": train_ops.rotary_frequencies(128, device=hip_device)} if turned else {}
    op = pick_attn_op(KsanaAttentionConfig(backend="sage_attention"))(num_heads=4, num_kv_heads=2, head_size=128, causal=True)
    one, two = (cache_ops.PagedCache(*(torch.zeros((2, 2, 16, 128), device=hip_device).to(kind) for _ in range(2))) for _ in range(2))
    o = op(q, k, v, kv_cache=one, pages=pages, k_lens=lens, **({"rotary": f} if turned else {}))
    x = [t.to(of) for t in (q, k, v)]
    if turned:
        x[0] = cache_ops.append(x[1], x[2], two, pages, lens, q=x[0], **f)
    else:
        cache_ops.append(x[1], x[2], two, pages, lens)
    want = cache_ops.attention(x[0], two, pages, lens, is_causal=True)
    assert o.dtype == torch.float32 and torch.equal(o, want.float())
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(one[:2], two[:2]))


def test_another_16_bit_type_is_refused(hip_device):
    x = torch.zeros((1, 2, 2, 128), dtype=torch.bfloat16, device=hip_device)
    op = pick_attn_op(KsanaAttentionConfig(backend="sage_attention"))(num_heads=2, head_size=128)
    with pytest.raises(ValueError, match="does not go with"):
        op(x, x, x, kv_cache=cache_ops.allocate(2, 16, 2, 128, torch.float16), pages=torch.zeros((1, 1), dtype=torch.int32, device=hip_device), k_lens=[2])
