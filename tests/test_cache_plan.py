"""Into how many runs the paged cache's attention cuts calls of few rows, from the scratch that it asks for; runs without a GPU."""

import ctypes as C

import pytest

from ksanadit_amd import _capi
from tests.test_cache_ops import _attn, _cache

HEADS, GROUP, PAGE = 8, 4, 64


def workgroups(sequences, tokens, D, dtype):
    nbytes = C.c_uint64(0)
    heads = HEADS * GROUP
    call = _attn(B=sequences, Hq=heads, Hkv=HEADS, Lq=1, D=D, q_strides=_capi.Strides(heads * D, heads * D, D, 1), o_strides=_capi.Strides(heads * D, heads * D, D, 1))
    cache = _cache(pages=4096, page_size=PAGE, table_width=-(-tokens // PAGE), strides=(C.c_int64 * 3)(HEADS * PAGE * D, PAGE * D, D), dtype=dtype)
    assert _capi.load().ksana_sage_cache_attn_scratch(C.addressof(call), C.addressof(cache), C.addressof(nbytes)) == 0
    return nbytes.value // (GROUP * (D + 2) * 4)  # a row's sums and a pair, of every run


@pytest.mark.parametrize("D,dtype,places", [(128, _capi.BF16, 512), (128, _capi.E4M3, 1024), (64, _capi.BF16, 1024), (64, _capi.E4M3, 1024)])
def test_one_round_of_workgroups(D, dtype, places):
    """Eight sequences of 4096 tokens fill the places that a compute unit's LDS and registers leave, once."""
    assert workgroups(8, 4096, D, dtype) == places
