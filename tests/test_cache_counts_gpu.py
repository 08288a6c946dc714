"""More tokens than a table has room for: the caller's error, which both calls stand, each as it is documented."""

import pytest
import torch

from ksanadit_amd import cache_ops, train_ops
from tests.test_cache_gpu import BF16, FP8, check_attention, pages_of
from tests.test_rotary_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, FP8])
@pytest.mark.parametrize("L,held", [(8, 35), (8, 32), (8, 40), (40, 41), (1, 33), (8, 2**31 - 1)])
def test_a_count_beyond_the_table_through_both_calls(hip_device, kind, L, held):
    page, room, D = 16, 32, 64
    g = torch.Generator().manual_seed(L)
    cache = cache_ops.PagedCache(*pages_of(4, 2, page, D, kind, hip_device, fill=0.5))
    before = [t.float().clone() for t in cache[:2]]
    wide = torch.tensor([[3, 1, 0, 2]], dtype=torch.int32, device=hip_device)
    table = wide[:, :2]  # (entries behind it are not read)
    q, k, v = (torch.randn((1, L, h, D), generator=g).to(hip_device, BF16) for h in (4, 2, 2))
    f = train_ops.rotary_frequencies(D, device=hip_device)
    counts = torch.tensor([held], dtype=torch.int32, device=hip_device)
    qr = cache_ops.append(k, v, cache, table, counts, q=q, frequencies=f)
    # append: rows at their own positions, those with a place are stored
    at = torch.arange(held - L, held, device=hip_device)[None]
    check(qr, q, f, at, None, True)
    kr = train_ops.rotary(k.float(), frequencies=f, positions=at)
    order = wide[0, : room // page].long()
    now = [t.float()[order].transpose(1, 2).reshape(room, 2, D) for t in cache[:2]]
    were = [t[order].transpose(1, 2).reshape(room, 2, D) for t in before]
    for stored, was, x in zip(now, were, (kr, v)):
        for t in range(room):
            i = t - (held - L)
            want = x[0, i].to(kind).float() if 0 <= i < L else was[t]
            # (a step of the type, where the turn's own rounding decides between two numbers)
            assert bool(((stored[t] - want).abs() <= want.abs() * 2.0**-2 + 2.0**-9 if kind == FP8 else (stored[t] - want).abs() <= want.abs() * 2.0**-7 + 2.0**-20).all()), t
    assert all(torch.equal(t.float()[i], b[i]) for t, b in zip(cache[:2], before) for i in (0, 2))
    # attention: the table's end is the sequence's
    o = cache_ops.attention(qr, cache, table, counts)
    last = min(L, room)
    check_attention(o[:, L - last :], qr[:, L - last :], [[t.double() for t in now]], [last], True)
    assert bool((o[:, : L - last] == 0).all())
