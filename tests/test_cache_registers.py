"""What the compiler made of the rotary step's and the paged cache's kernels, from the metadata in the built library; runs without a GPU."""

import pytest

from tests.test_registers import registers_in_memory  # noqa: F401  (a fixture)


@pytest.mark.parametrize("kernel,number,most", [("sage_rotary_kernel", 21, 5), ("sage_cache_rows_kernel", 8, 20), ("sage_cache_few_kernel", 8, 9), ("sage_cache_join_kernel", 8, 0)])
def test_registers_of_the_cache(registers_in_memory, kernel, number, most):  # noqa: F811
    """What goes through memory as they were measured, outside the attention's loops: not more."""
    found = {name: n for name, n in registers_in_memory.items() if kernel in name}
    assert len(found) == number
    assert max(found.values()) <= most, found
