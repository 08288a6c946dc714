"""Codes of 8-bit caches with scales: the nearest of the quotient, and of two as near the even one."""

import pytest
import torch

from ksanadit_amd import cache_ops

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def nearest(y):
    """e4m3's nearest number of float64 ones: 8 steps to a factor of two from 2^-6 on, 2^-9 apart below."""
    step = torch.exp2(torch.frexp(y)[1].double().clamp(min=-5) - 4)
    return (torch.round(y / step) * step).clamp(-448, 448)  # (torch.round: to even)


def test_the_tests_own_rounding():
    codes = torch.arange(0x7F, dtype=torch.uint8).view(FP8).double()
    assert torch.equal(nearest(codes), codes)
    between = (codes[:-1] + codes[1:]) / 2
    even = torch.where(torch.arange(0x7E) % 2 == 0, codes[:-1], codes[1:])
    assert torch.equal(nearest(between), even)
    assert torch.equal(nearest(between * (1 + 2.0**-40)), codes[1:]) and torch.equal(nearest(-between * (1 - 2.0**-40)), -codes[:-1])


def scales(numbers):
    """Of few bits, so that quotients lie between two codes; quotients next to such; next to nothing and next to fp32's largest."""
    few = [n * 2.0**-9 for n in (1, 3, 5, 7, 9, 11, 13, 15, 17, 19, 21, 23, 25, 27, 29, 31)]
    g = torch.Generator().manual_seed(5)
    between = (torch.arange(16, 31, dtype=torch.float64) + 0.5)[torch.randint(0, 15, (48,), generator=g)]
    x = numbers[torch.randint(0, numbers.numel(), (48,), generator=g)].double()
    near = (x / between).float()
    near = torch.cat((near, torch.nextafter(near, torch.tensor(0.0)), torch.nextafter(near, torch.tensor(torch.inf)))).tolist()
    return torch.tensor(few + near + [2.0**-149, 2.0**-140, 3 * 2.0**-130, 2.0**-126, 1.5 * 2.0**-127, 2.0**126, 1.7e38, 3.4e38], dtype=torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_are_the_nearest(hip_device, dtype):
    bits = torch.arange(2**15, dtype=torch.int32).to(torch.int16).view(dtype)
    some = bits[(bits.float() >= 2.0**-4) & (bits.float() < 4.0)]
    s = scales(some)
    every = bits[bits.isfinite()]
    g = torch.Generator().manual_seed(6)
    x = torch.cat((some[torch.randperm(some.numel(), generator=g)[:768]], every[torch.randperm(every.numel(), generator=g)[:1277]], torch.tensor([0.0, torch.inf, torch.nan], dtype=dtype)))
    x = torch.cat((x, -x)).reshape(1, -1, 1, 128).expand(1, 32, s.numel(), 128).to(hip_device)
    s = s.to(hip_device)
    cache = cache_ops.allocate(2, 16, s.numel(), 128, FP8, k_scale=s, v_scale=s)
    cache_ops.append(x, -x, cache, torch.tensor([[1, 0]], dtype=torch.int32, device=hip_device), [32])
    for t, y in zip(cache[:2], (x, -x)):
        got = t[[1, 0]].transpose(1, 2).reshape(32, s.numel(), 128).double()
        want = nearest(y[0].double() / s.double()[:, None])
        wrong = [int((a != b).sum()) for a, b in ((got.isnan(), want.isnan()), (got.nan_to_num(), want.nan_to_num()), (got.signbit() & ~got.isnan(), y[0].signbit() & ~y[0].isnan()))]
        assert wrong == [0, 0, 0]
