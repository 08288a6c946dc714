"""Sums over very many keys of the paged cache's attention."""

import math

import pytest
import torch

from ksanadit_amd import cache_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,kind", [(64, torch.float16), (128, torch.float16), (64, torch.float8_e4m3fn), (128, torch.float8_e4m3fn)])
def test_equal_weights_behind_a_larger_one(hip_device, monkeypatch, D, kind):
    """Key 0 has the weight 1 and all others the same one, whose additions one by one would all be rounded the same way: by 0.3 % of the sum in the end.

    Values are the same for all keys, so they are the result.  1999 / 2048 is an fp16 number, so that probabilities are off by nothing.  An addition is off by 2^-24 of the
    running sum, on average of half of the last one: of tiles of 64 keys in the sum of weights, of 16 keys in the products; exponentials, a tile's sum and factors 2^-20; the result half a step."""
    n, H, L, page = 8192 * 64, 8, 8192, 64
    taken = []
    monkeypatch.setattr(cache_ops, "_scratch", lambda nbytes, device: taken.append(nbytes))
    k = torch.zeros((n // page, 1, page, D), dtype=torch.float16, device=hip_device)
    k[0, 0, 0, 0] = 1.0
    values = torch.arange(1, D + 1, device=hip_device) / 8.0 if kind == torch.float16 else torch.arange(D, device=hip_device) % 8 / 4.0 + 2.0
    cache = cache_ops.PagedCache(k.to(kind), values.to(kind).expand(n // page, 1, page, D).contiguous())
    q = torch.zeros((1, L, H, D), dtype=torch.float16, device=hip_device)
    q[..., 0] = 1.0
    pages = torch.arange(n // page, dtype=torch.int32, device=hip_device)[None]
    o = cache_ops.attention(q, cache, pages, [n], is_causal=False, sm_scale=math.log(2048 / 1999))
    assert taken == [0]  # (512 blocks, none of them cut)
    want = values.to(kind).double()
    off = (o.double() - want).abs().amax((0, 1, 2)) / want
    print("off by", float(off.max()))
    assert bool((off <= 2.0**-11 + (n / 64 + n / 16) * 2.0**-25 + 2.0**-20).all()), float(off.max())
