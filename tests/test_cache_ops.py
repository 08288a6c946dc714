"""Rotary positions and the paged cache where no GPU is needed: what they refuse, frequencies, and the tests' own formula against differences."""

import ctypes as C
import math

import pytest
import torch

from ksanadit_amd import KsanaAttentionConfig, _capi, cache_ops, pick_attn_op, train_ops
from tests.test_rotary_gpu import turned

FAKE = 1 << 20  # an address that no call gets as far as using


# ------------------------------------------------------------------------------------------------ the formula
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("sections", [None, (4, 1, 3)])
def test_the_turn_against_its_definition(interleaved, sections):
    """Pair by pair, from cosines and sines."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn((2, 3, 2, 20), generator=g, dtype=torch.float64)
    f = train_ops.rotary_frequencies(16, sections=sections, device="cpu")
    at = torch.randint(-50, 50, (2, 3) if sections is None else (2, 3, 3), generator=g)
    y, _ = turned(x, f, at, sections, interleaved, 1.5)
    for b in range(2):
        for l in range(3):
            for i in range(8):
                axis = 0 if sections is None else (0 if i < 4 else 1 if i < 5 else 2)
                t = float(at[b, l] if sections is None else at[b, l, axis]) * float(f[i])
                c, d = (2 * i, 2 * i + 1) if interleaved else (i, i + 8)
                a, e = x[b, l, :, c], x[b, l, :, d]
                torch.testing.assert_close(y[b, l, :, c], 1.5 * (a * math.cos(t) - e * math.sin(t)), rtol=0, atol=1e-12)
                torch.testing.assert_close(y[b, l, :, d], 1.5 * (a * math.sin(t) + e * math.cos(t)), rtol=0, atol=1e-12)
    assert torch.equal(y[..., 16:], x[..., 16:])
    back, _ = turned(y, f, at, sections, interleaved, 1 / 1.5, -1.0)
    torch.testing.assert_close(back, x, rtol=0, atol=1e-12)


def test_the_gradient_is_the_turn_back():
    """Central differences of a linear map: exact but for 2^-52 of sums of 240 products, divided by the step."""
    g = torch.Generator().manual_seed(2)
    x, d, dy = (torch.randn((2, 3, 2, 20), generator=g, dtype=torch.float64) for _ in range(3))
    f, at = train_ops.rotary_frequencies(16, device="cpu"), torch.randint(-50, 50, (2, 3), generator=g)
    plus, minus = ((turned(x + s * d, f, at)[0] * dy).sum() for s in (0.5, -0.5))
    assert abs(plus - minus - (turned(dy, f, at, sign=-1.0)[0] * d).sum()) < 1e-11


# ------------------------------------------------------------------------------------------------ frequencies
def test_frequencies():
    make = lambda *a, **kw: train_ops.rotary_frequencies(*a, device="cpu", **kw).tolist()  # noqa: E731
    assert make(8) == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert make(12, sections=(2, 4, 0)) == pytest.approx([1.0, 0.01, 1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert make(8, 1e8, scaling="linear", factor=4) == pytest.approx([0.25, 2.5e-3, 2.5e-5, 2.5e-7], rel=1e-15)
    by_base = make(8, scaling="base", factor=8)
    assert by_base[0] == 1.0 and by_base[3] == pytest.approx(0.001 / 8, rel=1e-14)
    # turns over 1000 positions: 159, 15.9, 1.59, 0.159; kept from 32 on, divided up to 1
    share = (1000 * 0.1 / (2 * math.pi) - 1) / 31, (1000 * 0.01 / (2 * math.pi) - 1) / 31
    want = [1.0, 0.1 * share[0] + 0.025 * (1 - share[0]), 0.01 * share[1] + 0.0025 * (1 - share[1]), 0.00025]
    assert make(8, scaling="parts", factor=4, original_length=1000) == pytest.approx(want, rel=1e-14)
    assert make(2, scaling="base", factor=8) == [1.0]


@pytest.mark.parametrize("args,kw", [((7,), {}), ((0,), {}), ((8,), {"sections": (2, 3)}), ((8,), {"sections": (5, -1)}), ((8,), {"scaling": "cubic"}),
                                     ((8,), {"scaling": "linear", "factor": 0.0}), ((8,), {"scaling": "parts", "factor": 2.0}),
                                     ((8,), {"scaling": "parts", "factor": 2.0, "original_length": 9, "low": 3.0, "high": 2.0})])
def test_frequencies_that_are_refused(args, kw):
    with pytest.raises(ValueError):
        train_ops.rotary_frequencies(*args, device="cpu", **kw)


# ------------------------------------------------------------------------------------------------ refusals
def test_tensors_off_the_gpu_are_refused():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    cache, table = cache_ops.allocate(3, 16, 2, 64, device="cpu"), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: train_ops.rotary(q, frequencies=train_ops.rotary_frequencies(64, device="cpu")), lambda: cache_ops.attention(q, cache, table, [4]),
                 lambda: cache_ops.append(q, q, cache, table, [4])):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    for call in (lambda: train_ops.rotary(q[0], frequencies=None), lambda: cache_ops.attention(q[0], cache, table, [4]), lambda: cache_ops.append(q[0], q[0], cache, table, [4])):
        with pytest.raises(ValueError, match="4-D"):
            call()


def test_other_backends_refuse_a_cache():
    op = pick_attn_op(KsanaAttentionConfig(backend="torch_sdpa"))(num_heads=2, head_size=64)
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="kv_cache"):
        op(x, x, x, kv_cache=object())


def _rotary(**kw):
    c = _capi.Rotary(B=2, L=3, D=128, Hq=4, Hkv=2, dtype=_capi.BF16, width=128, interleaved=1, inverse=0, axes=1, ends=(C.c_int32 * 4)(64, 0, 0, 0), magnitude=1.0,
                     frequencies=FAKE, positions=None)
    for n, h in (("q_strides", 4), ("k_strides", 2), ("v_strides", 2)):
        setattr(c, n, _capi.Strides(3 * h * 128, h * 128, 128, 1))
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _cache(**kw):
    c = _capi.Cache(k=FAKE, v=FAKE, k_scale=None, v_scale=None, strides=(C.c_int64 * 3)(2 * 16 * 128, 16 * 128, 128), pages=9, page_size=16, dtype=_capi.BF16, table_width=5,
                    table=FAKE, table_stride=5, q_lens=None, k_lens=FAKE)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _attn(**kw):
    c = _capi.CacheAttn(B=2, Hq=4, Hkv=2, Lq=3, D=128, dtype=_capi.BF16, causal=1, sm_scale=0.1)
    c.q_strides = c.o_strides = _capi.Strides(3 * 4 * 128, 4 * 128, 128, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _ends(*n):
    return (C.c_int32 * 4)(*n)


ROTARY = [({"B": 0}, -1), ({"L": 0}, -1), ({"Hq": -1}, -1), ({"D": 514}, -2), ({"Hq": 70000}, -2), ({"B": 1 << 13, "L": 1 << 12}, -2), ({"dtype": 3}, -1), ({"width": 3}, -1),
          ({"width": 130}, -1), ({"axes": 0}, -1), ({"axes": 5}, -1), ({"ends": _ends(63)}, -1), ({"axes": 2, "ends": _ends(65, 64)}, -1), ({"frequencies": None}, -1),
          ({"frequencies": FAKE + 4}, -1), ({"positions": FAKE + 2}, -1), ({"positions": FAKE + 4, "positions_64": 1}, -1),
          ({"position_strides": (C.c_int64 * 3)(0, -1, 0)}, -1), ({"magnitude": float("nan")}, -1), ({"magnitude": float("inf")}, -1),
          ({"q_strides": _capi.Strides(1, 1, 1, 2)}, -1), ({"k_strides": _capi.Strides(1, -1, 1, 1)}, -1)]


@pytest.mark.parametrize("kw,rc", ROTARY)
def test_calls_of_the_rotary_step_are_checked(kw, rc):
    lib = _capi.load()
    assert lib.ksana_sage_rotary_rows(C.addressof(_rotary(**kw)), FAKE, FAKE, FAKE, FAKE, None) == rc, lib.ksana_sage_last_error()
    assert lib.ksana_sage_cache_append(C.addressof(_rotary(**kw)), C.addressof(_cache()), FAKE, FAKE, FAKE, FAKE, None) == rc, lib.ksana_sage_last_error()


def test_buffers_of_the_rotary_step_are_checked():
    lib, call, cache = _capi.load(), _rotary(), _cache()
    assert lib.ksana_sage_rotary_rows(None, FAKE, FAKE, FAKE, FAKE, None) == -1
    for i in range(4):
        for bad in (None, FAKE + 1, FAKE + 8):
            given = [FAKE] * 4
            given[i] = bad
            if i < 2 and bad == FAKE + 8:
                continue  # (rows are read at any address of their type)
            assert lib.ksana_sage_rotary_rows(C.addressof(call), *given, None) == -1
    for i in range(4):
        given = [FAKE] * 4
        given[i] = None
        assert lib.ksana_sage_cache_append(C.addressof(call), C.addressof(cache), *given, None) == -1
    assert lib.ksana_sage_cache_append(C.addressof(call), None, FAKE, FAKE, FAKE, FAKE, None) == -1
    assert lib.ksana_sage_cache_append(C.addressof(_rotary(dtype=_capi.FP32)), C.addressof(cache), FAKE, FAKE, FAKE, FAKE, None) == -1
    assert lib.ksana_sage_cache_append(C.addressof(_rotary(Hkv=0)), C.addressof(cache), FAKE, FAKE, FAKE, FAKE, None) == -1


def _strides(*n):
    return (C.c_int64 * 3)(*n)


CACHE = [({"pages": 0}, -1), ({"page_size": 0}, -1), ({"table_width": 0}, -1), ({"dtype": _capi.FP16}, -1), ({"k": None}, -1), ({"v": FAKE + 8}, -1), ({"table": None}, -1),
         ({"k_lens": None}, -1), ({"k_lens": FAKE + 2}, -1), ({"q_lens": FAKE + 1}, -1), ({"table": FAKE + 2}, -1), ({"k_scale": FAKE}, -1), ({"v_scale": FAKE}, -1),
         ({"dtype": _capi.E4M3, "k_scale": FAKE + 2}, -1), ({"strides": _strides(4096, 2048, 120)}, -1), ({"strides": _strides(4096, 2048, 132)}, -1),
         ({"strides": _strides(-4096, 2048, 128)}, -1), ({"table_stride": -1}, -1), ({"pages": 1 << 24, "page_size": 16}, -2), ({"page_size": 1 << 28}, -2),
         ({"strides": _strides(4096, 2048, 1 << 25)}, -2), ({"strides": _strides(1 << 35, 2048, 128), "pages": 1}, -2)]


@pytest.mark.parametrize("kw,rc", CACHE)
def test_caches_are_checked(kw, rc):
    lib, n = _capi.load(), C.c_uint64(0)
    cache = _cache(**kw)
    assert lib.ksana_sage_cache_attn_scratch(C.addressof(_attn()), C.addressof(cache), C.addressof(n)) == rc, lib.ksana_sage_last_error()
    assert lib.ksana_sage_cache_attn_fwd(C.addressof(_attn()), C.addressof(cache), FAKE, FAKE, FAKE, None) == rc
    assert lib.ksana_sage_cache_append(C.addressof(_rotary()), C.addressof(cache), FAKE, FAKE, FAKE, FAKE, None) == rc


@pytest.mark.parametrize("kw,rc", [({}, 0), ({"B": 0}, -1), ({"Lq": 0}, -1), ({"Hkv": 3}, -1), ({"D": 96}, -2), ({"dtype": 2}, -1), ({"sm_scale": float("nan")}, -1), ({"sm_scale": 3e38}, -1),
                                   ({"Lq": 1 << 25}, -2), ({"Hq": 2 << 10, "Lq": 1 << 20}, -2), ({"B": 1 << 20}, -2), ({"B": 1 << 17, "Lq": 1 << 20}, -2)])
def test_calls_of_the_attention_are_checked(kw, rc):
    lib, n = _capi.load(), C.c_uint64(0)
    assert lib.ksana_sage_cache_attn_scratch(C.addressof(_attn(**kw)), C.addressof(_cache()), C.addressof(n)) == rc, lib.ksana_sage_last_error()
    assert lib.ksana_sage_cache_attn_scratch(C.addressof(_attn()), C.addressof(_cache()), None) == -1
    assert lib.ksana_sage_cache_attn_scratch(None, C.addressof(_cache()), C.addressof(n)) == -1


def test_buffers_of_the_attention_are_checked():
    lib, call, cache, n = _capi.load(), _attn(), _cache(table_width=4096), C.c_uint64(0)
    assert lib.ksana_sage_cache_attn_scratch(C.addressof(call), C.addressof(cache), C.addressof(n)) == 0 and n.value > 0
    for q, o, scratch in ((None, FAKE, FAKE), (FAKE + 8, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE + 2, FAKE), (FAKE, FAKE, None), (FAKE, FAKE, FAKE + 128)):
        assert lib.ksana_sage_cache_attn_fwd(C.addressof(call), C.addressof(cache), q, o, scratch, None) == -1
    assert lib.ksana_sage_cache_attn_fwd(C.addressof(_attn(q_strides=_capi.Strides(3 * 4 * 128, 4 * 128, 124, 1))), C.addressof(cache), FAKE, FAKE, FAKE, None) == -1


def test_the_structures_are_packed_as_declared():
    for packed, declared in ((train_ops._ROTARY, _capi.Rotary), (cache_ops._CACHE, _capi.Cache), (cache_ops._ATTENTION, _capi.CacheAttn)):
        assert packed.size == C.sizeof(declared)


def test_pages_and_slots_of_tokens(tmp_path):
    """The kernels' division by a page's size, compiled for the host."""
    import re
    import subprocess
    from pathlib import Path

    header = (Path(_capi.__file__).parent / "csrc" / "sage_cache.h").read_text()
    body = re.search(r"struct Divisor \{.*?^__host__ __device__ inline int quotient.*?^\}", header, re.S | re.M).group(0).replace("__host__ __device__ ", "")
    source = tmp_path / "divide.cpp"
    source.write_text("#include <cstdint>\n#include <cstdio>\n#include <initializer_list>\n" + body + """
int main() {
  unsigned seed = 1;
  auto next = [&] { return seed = seed * 1664525u + 1013904223u; };
  long wrong = 0;
  for (int i = 0; i < 40000; ++i) {
    const int by = i < 5000 ? i + 1 : (int)(next() >> 1 >> (next() >> 27) | 1);
    const Divisor d = divisor(by);
    auto at = [&](int64_t x) { wrong += x >= 0 && x < (INT64_C(1) << 31) && quotient((int)x, d) != x / by; };
    const int64_t top = (INT64_C(1) << 31) / by * by;
    for (int64_t x : {INT64_C(0), (int64_t)by - 1, (int64_t)by, (int64_t)by + 1, top - 1, top, top - by - 1, (INT64_C(1) << 31) - 1}) at(x);
    for (int j = 0; j < 50; ++j) at(next() >> 1);
  }
  std::printf("%ld", wrong);
}
""")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(tmp_path / "divide"), str(source)], check=True)
    assert subprocess.run([str(tmp_path / "divide")], check=True, capture_output=True, text=True).stdout == "0"
