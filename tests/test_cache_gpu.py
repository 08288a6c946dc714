"""The paged cache on the GPU: what is stored, and attention on it, against dense definitions in 64 bits."""

import pytest
import torch

from ksanadit_amd import KsanaAttentionConfig, cache_ops, pick_attn_op, train_ops
from tests.test_rotary_gpu import turned

pytestmark = pytest.mark.gpu

BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
HALF_STEP = {BF16: 2.0**-8, FP16: 2.0**-11, FP8: 2.0**-4}


def tables(lens, page, device, seed=0, spare=3, wider=2):
    """Pages in no order for sequences of ``lens`` tokens, what lies behind a sequence's last page named by entries that name none."""
    g = torch.Generator().manual_seed(seed)
    needed = [-(-n // page) for n in lens]
    pages = sum(needed) + spare
    order = torch.randperm(pages, generator=g).tolist()
    rows, used = [], 0
    for i, n in enumerate(needed):
        rows.append(order[used : used + n] + [(-1, pages, 2**31 - 1, -(2**31))[(i + j) % 4] for j in range(max(needed) + wider - n)])
        used += n
    return torch.tensor(rows, dtype=torch.int32, device=device), pages


def pages_of(pages, heads, page, D, dtype, device, layout="heads first", fill=float("nan")):
    """Empty keys and values, laid out alike; what nothing is stored to is not a number."""
    def one():
        if layout == "heads first":
            t = torch.empty((pages, heads, page, D), dtype=dtype, device=device)
        elif layout == "slots first":
            t = torch.empty((pages, page, heads, D), dtype=dtype, device=device).transpose(1, 2)
        else:  # with room around rows and heads
            t = torch.empty((pages, heads + 1, page + 2, 2 * D), dtype=dtype, device=device)[:, 1:, 1 : page + 1, D:]
        t.copy_(torch.full((), fill, device=device))
        return t

    return one(), one()


def place(cache, table, b, t, page):
    return int(table[b, t // page]), t % page


def filled(lens, page, heads, D, dtype, device, layout="heads first", seed=0, scales=None, std=1.0):
    """(cache, table, keys and values of every sequence in 64 bits)"""
    table, pages = tables(lens, page, device, seed)
    k, v = pages_of(pages, heads, page, D, dtype, device, layout)
    g = torch.Generator().manual_seed(seed + 1)
    dense = []
    for b, n in enumerate(lens):
        own = []
        for t, scale in zip((k, v), scales or (None, None)):
            x = (torch.randn((n, heads, D), generator=g) * std).to(device)
            # (beyond 448 torch's cast gives not-a-numbers: nothing could be checked against those)
            x = (x if scale is None else x / scale[:, None])
            x = (x.clamp(-448, 448) if dtype == FP8 else x).to(dtype)
            at = torch.arange(n, device=device)
            raw = t.view(torch.uint8) if dtype == FP8 else t
            if n:
                raw[table[b].long()[at // page], :, at % page] = x.view(torch.uint8) if dtype == FP8 else x
            own.append(x.float().double() if scale is None else x.float().double() * scale.double()[:, None])
        dense.append(own)
    return cache_ops.PagedCache(k, v, *(scales or (None, None))), table, dense


def check_attention(o, q, dense, new, causal, sm_scale=None, hidden=None, parts=1):
    """Against the definition; off by
    - half a step of q's type of every weight where it is multiplied on (its square where that is done in two parts), and of the result;
    - fp32's: a score of D products and sums, by its terms' sizes (D + 8) 2^-24, counted twice in the normalised weight, and 2^-20 for exponentials, sums and factors;
    - in fp16, weights that are subnormal: 2^-31 of the row's largest each."""
    B, L, H, D = q.shape
    half = HALF_STEP[q.dtype]
    scale = D**-0.5 if sm_scale is None else sm_scale
    worst = 0.0
    for b in range(B):
        n = dense[b][0].shape[0]
        m = min(new[b], L)
        assert bool((o[b, m:] == 0).all()), "rows behind the counts"
        if m == 0:
            continue
        k, v = (t.repeat_interleave(H // t.shape[1], 1).transpose(0, 1) for t in dense[b])  # [H, n, D]
        x = q[b, :m].double().transpose(0, 1)
        s = x @ k.transpose(1, 2) * scale
        size = (x.abs() @ k.abs().transpose(1, 2) * abs(scale)) if n else s
        seen = torch.ones((m, n), dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(n, device=q.device)[None] <= torch.arange(n - m, n, device=q.device)[:, None]
        if hidden is not None:
            seen = seen & ~hidden[b][None, :n]
        s = s.masked_fill(~seen, -torch.inf)
        w = torch.softmax(s, -1).nan_to_num(0.0)
        want = w @ v
        ds = size.masked_fill(~seen, 0.0).amax(-1, keepdim=True) * (D + 8) * 2.0**-24 if n else torch.zeros((H, m, 1), device=q.device)
        weighed = w @ v.abs()
        largest = v.abs().amax(1, keepdim=True) if n else torch.zeros_like(want)
        bound = (half**parts + 2 * ds + 2.0**-20) * weighed + half * want.abs() + n * 2.0**-31 * largest * (q.dtype == FP16) + torch.finfo(q.dtype).smallest_normal * half * 2
        off = (o[b, :m].double().transpose(0, 1) - want).abs()
        worst = max(worst, float((off / bound).max()))
        assert bool((off <= bound).all()), (b, float((off / bound).max()), off.isnan().sum())
    return worst


ATTENTION = [
    # tokens, new ones, heads, key heads, D, page, causal, dtype, cache, layout
    ([1], [1], 1, 1, 128, 16, True, BF16, BF16, "heads first"),
    ([1], [1], 8, 1, 64, 1, True, FP16, FP16, "heads first"),
    ([63, 64, 65, 1], [1, 1, 1, 1], 8, 2, 128, 16, True, BF16, BF16, "slots first"),
    ([300, 5, 0, 129], [7, 5, 0, 1], 4, 4, 64, 20, True, FP16, FP16, "heads first"),
    ([300, 5, 0, 129], [7, 5, 0, 1], 10, 2, 128, 7, False, BF16, BF16, "room"),
    ([257, 130], [257, 130], 2, 1, 128, 64, True, BF16, BF16, "heads first"),
    ([1000, 200], [130, 129], 6, 2, 64, 128, True, FP16, FP16, "slots first"),
    ([1000, 200], [130, 129], 5, 1, 128, 100, True, FP16, FP8, "heads first"),
    ([640, 64], [64, 64], 3, 3, 128, 64, True, BF16, FP8, "room"),
    ([640, 64], [64, 0], 3, 3, 64, 32, False, BF16, FP8, "slots first"),
    ([5000], [1], 40, 8, 128, 64, True, BF16, BF16, "heads first"),
    ([5000], [3], 40, 8, 128, 16, True, BF16, FP8, "heads first"),
    ([4097, 31, 2048], [1, 1, 1], 16, 16, 64, 16, True, FP16, FP16, "heads first"),
    ([3000], [33], 32, 1, 128, 256, True, BF16, BF16, "heads first"),
    ([700], [5], 7, 1, 128, 1560, True, BF16, BF16, "heads first"),
    ([1561, 3], [1560, 3], 1, 1, 128, 1560, False, FP16, FP16, "heads first"),
    ([2000], [1664], 40, 8, 64, 100, True, BF16, BF16, "heads first"),  # more blocks than fill a round: the last ones cut
    ([2000], [1664], 40, 8, 128, 100, False, FP16, FP16, "slots first"),
    ([2300, 900], [4, 4], 8, 1, 128, 65, True, BF16, BF16, "heads first"),  # 32 rows
    ([2300, 900], [11, 3], 3, 1, 64, 63, True, BF16, FP8, "heads first"),  # 33 rows
]


@pytest.mark.parametrize("lens,new,H,Hkv,D,page,causal,dtype,kind,layout", ATTENTION)
def test_attention(hip_device, lens, new, H, Hkv, D, page, causal, dtype, kind, layout):
    scales = None
    if kind == FP8:
        scales = [torch.linspace(0.005, 0.02, Hkv, device=hip_device) for _ in range(2)]
    cache, table, dense = filled(lens, page, Hkv, D, kind, hip_device, layout, seed=D + H, scales=scales)
    L = max(max(new), 1) + (2 if len(lens) > 1 else 0)
    q = torch.randn((len(lens), L, H, D), generator=torch.Generator().manual_seed(9)).to(hip_device, dtype)
    for b, n in enumerate(new):
        q[b, n:] = float("nan")  # (not read)
    counts = [torch.tensor(n, dtype=torch.int32, device=hip_device) for n in (lens, new)]
    o = cache_ops.attention(q, cache, table, *counts, is_causal=causal)
    print("share of the bound", check_attention(o, q, dense, new, causal))
    assert torch.equal(o, cache_ops.attention(q, cache, table, lens, new, is_causal=causal))
    if L == new[0] and len(lens) == 1:
        assert torch.equal(o, cache_ops.attention(q, cache, table, counts[0], is_causal=causal))


@pytest.mark.parametrize("lens,new,H,Hkv,D,page,dtype", [([5000, 77], [1, 1], 40, 8, 128, 16, BF16), ([700, 3, 0], [4, 3, 0], 8, 1, 64, 64, FP16), ([129], [32], 2, 2, 128, 20, BF16)])
def test_few_rows_are_rounded_once(hip_device, lens, new, H, Hkv, D, page, dtype):
    """On 16-bit caches: their probabilities are multiplied on in two parts."""
    cache, table, dense = filled(lens, page, Hkv, D, dtype, hip_device)
    q = torch.randn((len(lens), max(new), H, D), generator=torch.Generator().manual_seed(2)).to(hip_device, dtype)
    check_attention(cache_ops.attention(q, cache, table, lens, new), q, dense, new, True, parts=2)


@pytest.mark.parametrize("sm_scale", [0.0, -0.3, 3.0])
def test_scales(hip_device, sm_scale):
    cache, table, dense = filled([200], 16, 2, 64, BF16, hip_device)
    q = torch.randn(1, 3, 4, 64, device=hip_device).bfloat16()
    check_attention(cache_ops.attention(q, cache, table, [200], sm_scale=sm_scale), q, dense, [3], True, sm_scale)


@pytest.mark.parametrize("Lq,page", [(1, 16), (1, 64), (40, 16), (200, 64), (200, 24)])
@pytest.mark.parametrize("kind", [BF16, FP8])
def test_pages_that_do_not_exist_are_not_seen(hip_device, Lq, page, kind):
    lens = [500, 500]
    cache, table, dense = filled(lens, page, 2, 128, kind, hip_device)
    hidden = torch.zeros((2, 500), dtype=torch.bool, device=hip_device)
    for b, i, entry in ((0, 0, -1), (0, 2, cache.k.shape[0]), (1, 3, 2**31 - 1), (1, 499 // page, -7)):
        table[b, i] = entry
        hidden[b, i * page : (i + 1) * page] = True
    q = torch.randn((2, Lq, 4, 128), device=hip_device).bfloat16()
    o = cache_ops.attention(q, cache, table, lens)
    check_attention(o, q, dense, [Lq, Lq], True, hidden=hidden)
    table.fill_(-1)
    assert bool((cache_ops.attention(q, cache, table, lens) == 0).all())


def test_counts_that_do_not_fit(hip_device):
    """Clamped to the table and the rows; more new tokens than there are: the rows before the sequence's start see nothing."""
    cache, table, dense = filled([100], 16, 1, 64, BF16, hip_device)
    table = table[:, :7]
    q = torch.randn(1, 8, 1, 64, device=hip_device).bfloat16()
    short = [[t[:5] for t in dense[0]]]
    o = cache_ops.attention(q, cache, table, [5], [8])
    assert bool((o[:, :3] == 0).all())
    check_attention(o[:, 3:], q[:, 3:], short, [5], True)
    for k_lens, q_lens in (([-3], [4]), ([0], [8]), ([50], [0]), ([50], [-2])):
        assert bool((cache_ops.attention(q, cache, table, k_lens, q_lens) == 0).all())
    cache.k[:, :, 100 - 96 :][int(table[0, 6])] = 0.0  # (the last page's slots behind the sequence: a count beyond the table sees them)
    cache.v[:, :, 100 - 96 :][int(table[0, 6])] = 0.0
    longer = [[torch.cat((t, t.new_zeros(12, 1, 64))) for t in dense[0]]]
    check_attention(cache_ops.attention(q, cache, table, [2**31 - 1], [2**31 - 1]), q, longer, [8], True)


def test_sequences_may_share_pages(hip_device):
    cache, table, dense = filled([128, 128], 32, 2, 64, BF16, hip_device)
    table[1, :2] = table[0, :2]
    dense[1] = [torch.cat((a[:64], b[64:])) for a, b in zip(dense[0], dense[1])]
    q = torch.randn(2, 1, 2, 64, device=hip_device).bfloat16()
    check_attention(cache_ops.attention(q, cache, table, [128, 100]), q, [dense[0], [t[:100] for t in dense[1]]], [1, 1], True)


def test_weights_that_peak_and_values_that_are_no_numbers(hip_device):
    cache, table, dense = filled([300], 16, 1, 128, BF16, hip_device, std=6.0)
    q = (torch.randn(1, 2, 2, 128, device=hip_device) * 6).bfloat16()
    check_attention(cache_ops.attention(q, cache, table, [300]), q, dense, [2], True)
    p, s = place(cache, table, 0, 299, 16)
    cache.v[p, 0, s, 5] = float("nan")
    o = cache_ops.attention(q, cache, table, [300], is_causal=False)
    assert bool(o[..., 5].isnan().all()) and bool(o[..., 6:].isfinite().all())
    cache.k[p, 0, s, 5] = float("nan")
    assert bool(cache_ops.attention(q, cache, table, [300], is_causal=False).isnan().all())


def test_a_cache_beyond_32_bits(hip_device):
    """Pages whose offsets pass 2^32 bytes."""
    page, Hkv, D, pages = 128, 8, 128, 20000
    k, v = (torch.empty((pages, Hkv, page, D), dtype=BF16, device=hip_device) for _ in range(2))
    cache, small = cache_ops.PagedCache(k, v), filled([400], page, Hkv, D, BF16, hip_device)
    far = torch.tensor([[pages - 1, 3, pages - 700, 16384]], dtype=torch.int32, device=hip_device)
    for t, s in ((k, small[0].k), (v, small[0].v)):
        t[far[0].long()] = s[small[1][0, :4].long()]
    q = torch.randn(1, 2, 16, D, device=hip_device).bfloat16()
    check_attention(cache_ops.attention(q, cache, far, [400]), q, small[2], [2], True)
    new = torch.randn(1, 2, Hkv, D, device=hip_device).bfloat16()
    cache_ops.append(new, -new, cache, far, [402])
    assert torch.equal(k[16384, :, 16:18].transpose(0, 1), new[0]) and torch.equal(v[16384, :, 16:18].transpose(0, 1), -new[0])


# ------------------------------------------------------------------------------------------------ append

APPEND = [
    # tokens with the new ones, new ones, L, heads of q, key heads, D, page, width, interleaved, sections, dtype, cache, layout
    ([1], [1], 1, 2, 2, 128, 16, 128, True, None, BF16, BF16, "heads first"),
    ([40, 3, 0, 17], [5, 3, 0, 1], 6, 8, 2, 128, 16, 128, False, None, BF16, BF16, "slots first"),
    ([40, 3, 0, 17], [5, 3, 0, 1], 6, 5, 1, 64, 7, 32, True, None, FP16, FP16, "room"),
    ([1700, 1560], [1560, 1560], 1560, 3, 3, 128, 1560, 128, True, (22, 21, 21), BF16, FP8, "heads first"),
    ([200, 130], [130, 130], 130, 0, 4, 64, 64, 64, False, (10, 22), FP16, FP8, "slots first"),
    ([9, 9], [2, 9], 9, 0, 3, 128, 1, 0, True, None, BF16, BF16, "heads first"),
    ([9, 9], [2, 9], 9, 0, 3, 128, 5, 0, True, None, BF16, FP8, "heads first"),
    ([30], [20], 20, 4, 1, 64, 16, 20, False, None, FP16, FP16, "room"),  # halves of ten: value by value
    ([30], [20], 20, 4, 1, 64, 16, 12, True, None, BF16, FP8, "heads first"),
]


@pytest.mark.parametrize("lens,new,L,H,Hkv,D,page,width,interleaved,sections,dtype,kind,layout", APPEND)
def test_append(hip_device, lens, new, L, H, Hkv, D, page, width, interleaved, sections, dtype, kind, layout):
    B = len(lens)
    scales = [torch.linspace(0.01, 0.005, Hkv, device=hip_device), torch.linspace(0.004, 0.008, Hkv, device=hip_device)] if kind == FP8 else (None, None)
    table, pages = tables(lens, page, hip_device)
    store = pages_of(pages, Hkv, page, D, kind, hip_device, layout, fill=3.0)
    cache = cache_ops.PagedCache(*store, *scales)
    g = torch.Generator().manual_seed(4)
    rows = {n: torch.randn((B, L, h, D), generator=g).to(hip_device, dtype) for n, h in (("q", H), ("k", Hkv), ("v", Hkv)) if h}
    f = train_ops.rotary_frequencies(width, sections=sections, device=hip_device) if width else None
    positions = torch.randint(0, 1000, (B, L, len(sections)), generator=g).to(hip_device) if sections else None
    out = cache_ops.append(rows["k"], rows["v"], cache, table, lens, new, q=rows.get("q"), frequencies=f, positions=positions, sections=sections, interleaved=interleaved)
    at = torch.arange(L, device=hip_device)[None] + (torch.tensor(lens) - torch.tensor(new)).to(hip_device)[:, None]
    at = at if positions is None else positions

    def bound(y, size):  # (see test_rotary_gpu.check; the scale's inverse and the product besides)
        return size * 12 * 2.0**-24 + y.abs() * 2.0**-22

    def turn(x):
        return turned(x, f, at, sections, interleaved) if width else (x.double(), torch.zeros_like(x, dtype=torch.float64))

    if H:
        y, size = turn(rows["q"])
        for b in range(B):
            assert bool((out[b, new[b] :] == 0).all())
            off = (out[b, : new[b]].double() - y[b, : new[b]]).abs()
            assert bool((off <= y[b, : new[b]].abs() * HALF_STEP[dtype] + bound(y, size)[b, : new[b]] + 2.0**-24).all())
    else:
        assert out is None
    k, k_size = turn(rows["k"])
    v = rows["v"].double()
    touched = [torch.zeros(t.shape[:3], dtype=torch.bool, device=hip_device) for t in store]
    for t, y, size, scale, mark in zip(store, (k, v), (k_size, torch.zeros_like(v)), scales, touched):
        for b in range(B):
            for i in range(new[b]):
                p, s = place(cache, table, b, lens[b] - new[b] + i, page)
                mark[p, :, s] = True
                got, want, room = t[p, :, s].float().double(), y[b, i], bound(y, size)[b, i]
                if scale is not None:
                    want, room = want / scale.double()[:, None], room / scale.double()[:, None]
                    want = want.clamp(-448, 448)
                # (e4m3: normal numbers from 2^-6 on, the others 2^-9 apart)
                assert bool(((got - want).abs() <= want.abs() * HALF_STEP[kind] + room + (2.0**-10 if kind == FP8 else 2.0**-25)).all())
        assert bool((t.float()[~mark] == 3.0).all()), "slots that nothing was stored to"


def test_append_saturates_and_keeps_not_a_numbers(hip_device):
    cache = cache_ops.PagedCache(*pages_of(2, 1, 4, 64, FP8, hip_device, fill=0.0), torch.tensor([0.5], device=hip_device), None)
    k = torch.zeros((1, 1, 1, 64), dtype=BF16, device=hip_device)
    k[0, 0, 0, :6] = torch.tensor([1000.0, -1000.0, float("inf"), float("nan"), 224.0, 0.25])
    cache_ops.append(k, k, cache, torch.tensor([[1, -1]], dtype=torch.int32, device=hip_device), [1])
    first = cache.k[1, 0, 0, :6].float().tolist()
    assert first[:3] == [448.0, -448.0, 448.0] and first[3] != first[3] and first[4:] == [448.0, 0.5]
    assert cache.v[1, 0, 0, 4:6].float().tolist() == [224.0, 0.25]


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_every_code_of_an_8_bit_cache(hip_device, dtype):
    """Codes are what torch's cast gives, for every 16-bit number there is; values come back as they stand, for every code there is (one key: its weight is 1)."""
    numbers = torch.arange(-(2**15), 2**15, device=hip_device).short().view(dtype).reshape(1, 256, 2, 128)
    cache = cache_ops.PagedCache(*pages_of(16, 2, 16, 128, FP8, hip_device, fill=0.0))
    table = torch.arange(16, dtype=torch.int32, device=hip_device)[None]
    cache_ops.append(numbers, -numbers, cache, table, [256])
    for t, x in zip(cache[:2], (numbers, -numbers)):
        want = x[0].float().clamp(-448, 448).to(FP8).float()
        got = t.transpose(1, 2).reshape(256, 2, 128).float()
        assert torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(got.isnan(), x[0].isnan())
    codes = torch.arange(256, device=hip_device).to(torch.uint8).reshape(2, 1, 1, 128)
    v = codes.clone().view(FP8)
    one = cache_ops.PagedCache(torch.zeros_like(codes).view(FP8), v, None, torch.tensor([0.5], device=hip_device))
    for L in (1, 40):
        o = cache_ops.attention(torch.ones((2, L, 1, 128), dtype=dtype, device=hip_device), one, torch.tensor([[0], [1]], dtype=torch.int32, device=hip_device), [1, 1], is_causal=False)
        want = (v.float().reshape(2, 1, 1, 128) * 0.5).expand(2, L, 1, 128)
        assert torch.equal(o.float().nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(o.isnan(), want.isnan())


@pytest.mark.parametrize("L", [1, 40])
@pytest.mark.parametrize("kind", [BF16, FP8])
def test_keys_of_many_sizes(hip_device, L, kind):
    """A query picks one channel of every key: small and subnormal codes, and large ones, come into the scores as they are."""
    n = 127
    k = torch.zeros((n, 1, 1, 64), dtype=torch.uint8, device=hip_device)
    k[:, 0, 0, 3] = torch.arange(n, device=hip_device).to(torch.uint8)
    k = k.view(FP8)
    cache = cache_ops.PagedCache(*(t.to(kind) if kind != FP8 else t for t in (k, torch.randn((n, 1, 1, 64), device=hip_device).clamp(-4, 4).to(FP8))))
    q = torch.zeros((1, L, 1, 64), dtype=BF16, device=hip_device)
    q[..., 3] = torch.linspace(-0.25, 0.25, L, device=hip_device)[None, :, None] if L > 1 else 0.125
    table = torch.arange(n, dtype=torch.int32, device=hip_device)[None]
    dense = [[t.float().double().reshape(n, 1, 64) for t in cache[:2]]]
    check_attention(cache_ops.attention(q, cache, table, [n], is_causal=False, sm_scale=1.0), q, dense, [L], False, 1.0)


def test_append_stores_nothing_where_there_is_no_page(hip_device):
    cache = cache_ops.PagedCache(*pages_of(3, 1, 4, 64, BF16, hip_device, fill=7.0))
    k = torch.ones((4, 6, 1, 64), dtype=BF16, device=hip_device)
    table = torch.tensor([[0, 3], [-1, 1], [-(2**31), 2**31 - 1], [2, -1]], dtype=torch.int32, device=hip_device)
    # six rows each: of sequence 0 tokens 0 .. 5; of 1 likewise; 2; of 3 tokens 8 .. 13 behind the table, then before its start
    cache_ops.append(k, 2 * k, cache, table, [6, 6, 6, 14])
    for t, x in ((cache.k, 1.0), (cache.v, 2.0)):
        assert bool((t[0] == x).all()) and bool((t[1, :, :2] == x).all()) and bool((t[1, :, 2:] == 7).all()) and bool((t[2] == 7).all())
    cache_ops.append(k, k, cache, table, [0, -5, 2**31 - 1, 2], [-1, 6, 6, 6])
    assert bool((cache.k[2, :, :2] == 1).all()) and bool((cache.k[2, :, 2:] == 7).all())


# ------------------------------------------------------------------------------------------------ together

def _steps(device, kind, dtype, causal, chunks, H=8, Hkv=2, D=128, page=20):
    """Chunks of two sequences through a cache, each chunk's result; and all tokens' q, k and v."""
    g = torch.Generator().manual_seed(11)
    total = sum(chunks)
    q, k, v = (torch.randn((2, total, h, D), generator=g).to(device, dtype) for h in (H, Hkv, Hkv))
    table, pages = tables([total, total], page, device)
    scales = [torch.full((Hkv,), 0.01, device=device) for _ in range(2)] if kind == FP8 else (None, None)
    cache = cache_ops.PagedCache(*pages_of(pages, Hkv, page, D, kind, device), *scales)
    f = train_ops.rotary_frequencies(D, device=device)
    out, done = [], 0
    op = pick_attn_op(KsanaAttentionConfig(backend="sage_attention"))(num_heads=H, num_kv_heads=Hkv, head_size=D, causal=causal)
    for n in chunks:
        lens = torch.full((2,), done + n, dtype=torch.int32, device=device)
        part = [t[:, done : done + n] for t in (q, k, v)]
        out.append(op(*part, kv_cache=cache, pages=table, k_lens=lens, rotary={"frequencies": f, "interleaved": False}))
        done += n
    return torch.cat(out, 1), q, k, v, f, cache, table


@pytest.mark.parametrize("chunks", [[50, 1, 1, 1], [1, 130, 7], [64, 64, 64]])
def test_chunks_are_what_a_whole_sequence_is(hip_device, chunks):
    o, q, k, v, f, _, _ = _steps(hip_device, BF16, BF16, True, chunks)
    qr, kr = train_ops.rotary(q, k, frequencies=f, interleaved=False)
    want = train_ops.attention(qr, kr, v, is_causal=True)
    dense = [[kr[b].double(), v[b].double()] for b in range(2)]
    check_attention(o, qr, dense, [q.shape[1]] * 2, True)
    assert float((o.double() - want.double()).norm() / want.double().norm()) < 2 * 2.0**-8


def test_chunks_through_an_8_bit_cache(hip_device):
    """The result is attention on what the cache holds."""
    o, q, k, v, f, cache, table = _steps(hip_device, FP8, BF16, True, [40, 1, 90])
    qr = train_ops.rotary(q, frequencies=f, interleaved=False)
    total, page = q.shape[1], cache.k.shape[2]
    at = torch.arange(total, device=hip_device)
    raw = [t.view(torch.uint8) for t in cache[:2]]
    dense = [[r[table[b].long()[at // page], :, at % page].view(FP8).float().double() * 0.01 for r in raw] for b in range(2)]
    check_attention(o[:, 41:], qr[:, 41:], [[(t.float() * 1).double() for t in d] for d in dense], [90, 90], True)


def test_a_decoding_step_in_a_graph(hip_device):
    """Captured once; replays go by the counts, the table and the rows as they are then."""
    H, Hkv, D, page, B = 8, 2, 128, 16, 3
    table, pages = tables([400] * B, page, hip_device)
    f = train_ops.rotary_frequencies(D, device=hip_device)
    make = lambda: cache_ops.PagedCache(*pages_of(pages, Hkv, page, D, BF16, hip_device, fill=0.25))  # noqa: E731
    cache, other = make(), make()
    lens = torch.tensor([390, 1, 200], dtype=torch.int32, device=hip_device)
    q, k, v = (torch.zeros((B, 1, h, D), dtype=BF16, device=hip_device) for h in (H, Hkv, Hkv))

    def step(cache):
        return cache_ops.attention(cache_ops.append(k, v, cache, table, lens, q=q, frequencies=f), cache, table, lens)

    step(cache), step(other)  # (the warm-up stores rows too)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(cache)
    with torch.cuda.graph(second):
        twice = step(cache)
    for i in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(BF16))
        lens += torch.tensor([1, 1, 40], dtype=torch.int32, device=hip_device)
        (graph if i % 2 == 0 else second).replay()
        want = step(other)
        torch.cuda.synchronize()
        assert torch.equal(held if i % 2 == 0 else twice, want)
        assert torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)


def test_streams(hip_device):
    """Calls on two streams at once, each with scratch of its own."""
    cache, table, dense = filled([5000, 3000], 16, 8, 128, BF16, hip_device)
    qs = [torch.randn((2, 1, 40, 128), device=hip_device).bfloat16() for _ in range(4)]
    want = [cache_ops.attention(q, cache, table, [5000, 3000]) for q in qs]
    lens = torch.tensor([5000, 3000], dtype=torch.int32, device=hip_device)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cache_ops.attention(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_backends_without_a_cache_refuse_one(hip_device):
    x = torch.zeros((1, 2, 2, 128), dtype=BF16, device=hip_device)
    cache = cache_ops.allocate(2, 16, 2, 128)
    op = pick_attn_op(KsanaAttentionConfig(backend="torch_sdpa"))(num_heads=2, head_size=128)
    with pytest.raises(ValueError, match="kv_cache"):
        op(x, x, x, kv_cache=cache, pages=torch.zeros((1, 1), dtype=torch.int32, device=hip_device), k_lens=[2])


def test_refusals(hip_device):
    cache, table, _ = filled([40], 16, 2, 64, BF16, hip_device)
    q, k = torch.zeros((1, 3, 4, 64), dtype=BF16, device=hip_device), torch.zeros((1, 3, 2, 64), dtype=BF16, device=hip_device)
    f = train_ops.rotary_frequencies(64, device=hip_device)
    one = torch.ones(2, device=hip_device)
    bad = [
        (cache._replace(v=cache.v[:-1]), "laid out alike"), (cache._replace(v=cache.v.half()), "laid out alike"), (cache._replace(v=cache.v.cpu()), "laid out alike"),
        (cache._replace(k=cache.k.half(), v=cache.v.half()), "does not go with"), (cache._replace(k_scale=one), "k_scale"),
        (cache_ops.allocate(3, 16, 2, 128), "channels"), (cache_ops.allocate(0, 16, 2, 64), "empty"),
        (cache_ops.allocate(3, 16, 2, 64, FP8, k_scale=one[:1]), "k_scale"), (cache_ops.allocate(3, 16, 2, 64, FP8, v_scale=one.double()), "v_scale"),
        (cache_ops.PagedCache(*(torch.zeros(3, 2, 16, 128, dtype=BF16, device=hip_device)[..., ::2] for _ in range(2))), "contiguous"),
    ]
    for c, what in bad:
        with pytest.raises(ValueError, match=what):
            cache_ops.attention(q, c, table, [40])
        with pytest.raises(ValueError, match=what):
            cache_ops.append(k, k, c, table, [40])
    for t in (table.long(), table[0], table.cpu(), table[:, :0], table.expand(2, -1), torch.stack((table, table), -1)[..., 0]):
        with pytest.raises(ValueError, match="pages must be"):
            cache_ops.attention(q, cache, t, [40])
    with pytest.raises(ValueError, match="multiple of 16 bytes"):  # rows closer than their channels
        cache_ops.attention(q, cache_ops.PagedCache(*(torch.zeros(9999, dtype=BF16, device=hip_device).as_strided((3, 2, 16, 64), (2048, 1024, 56, 1)) for _ in range(2))), table, [40])
    for kw, what in (({"k_lens": None}, "k_lens"), ({"k_lens": [1, 2]}, "k_lens"), ({"q_lens": [1, 2]}, "q_lens"), ({"sm_scale": float("nan")}, "sm_scale"),
                     ({"q": q[:, :, :3]}, "no multiple"), ({"q": q[0]}, "4-D"), ({"q": q.float()}, "bfloat16 or float16")):
        with pytest.raises(ValueError, match=what):
            cache_ops.attention(**{"q": q, "cache": cache, "pages": table, "k_lens": [40], **kw})
    for kw, what in (({"v": k[:, :2]}, "incompatible"), ({"q": q}, "go with frequencies"), ({"positions": torch.zeros(3)}, "go with frequencies"),
                     ({"k": k[:, :, :1], "v": k[:, :, :1]}, "heads"), ({"frequencies": f.float()}, "float64"), ({"magnitude": float("nan")}, "magnitude")):
        with pytest.raises(ValueError, match=what):
            cache_ops.append(**{"k": k, "v": k, "cache": cache, "pages": table, "k_lens": [40], **kw})
    with pytest.raises(RuntimeError, match="no backward pass"):
        cache_ops.attention(q.clone().requires_grad_(), cache, table, [40])
    with pytest.raises(RuntimeError, match="no backward pass"):
        cache_ops.append(k, k.clone().requires_grad_(), cache, table, [40])
    with torch.no_grad():
        cache_ops.attention(q.clone().requires_grad_(), cache, table, [40])


def test_a_compiled_function_calls_it(hip_device):
    """The kernels are no operators of torch: a compiled function leaves its graph for them, in every call."""
    cache, table, dense = filled([40], 16, 2, 64, BF16, hip_device)
    f, lens = train_ops.rotary_frequencies(64, device=hip_device), torch.tensor([40], dtype=torch.int32, device=hip_device)
    q, k = torch.randn(1, 3, 4, 64, device=hip_device).bfloat16(), torch.randn(1, 3, 2, 64, device=hip_device).bfloat16()

    def step(q, k, cache):
        return cache_ops.attention(cache_ops.append(k, k * 2, cache, table, lens, q=q + 1, frequencies=f), cache, table, lens) * 2

    compiled = torch.compile(step, backend="aot_eager")
    for i in range(3):
        assert torch.equal(compiled(q + i, k, cache), step(q + i, k, cache))


def test_autograd_notices_writes(hip_device):
    cache, table, _ = filled([40], 16, 2, 64, BF16, hip_device)
    k = torch.zeros((1, 1, 2, 64), dtype=BF16, device=hip_device)
    x = torch.ones_like(cache.k, requires_grad=True)
    y = (x * cache.k).nan_to_num().sum()
    cache_ops.append(k, k, cache, table, [40])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        own = cache_ops.allocate(3, 16, 2, 64)
        cache_ops.append(k, k, own, table, [40])
    with pytest.raises(ValueError, match="require gradients"):
        cache_ops.append(k, k, cache._replace(k=cache.k.clone().requires_grad_()), table, [40])


def test_nothing_to_do(hip_device):
    cache, table, _ = filled([40], 16, 2, 64, BF16, hip_device)
    for shape in ((1, 0, 4, 64), (1, 3, 0, 64)):
        q = torch.zeros(shape, dtype=BF16, device=hip_device)
        assert cache_ops.attention(q, cache, table, [40]).shape == q.shape
    k = torch.zeros((1, 0, 2, 64), dtype=BF16, device=hip_device)
    q = torch.zeros((1, 0, 4, 64), dtype=BF16, device=hip_device)
    assert cache_ops.append(k, k, cache, table, [40]) is None
    assert cache_ops.append(k, k, cache, table, [40], q=q, frequencies=train_ops.rotary_frequencies(64, device=hip_device)).shape == q.shape
