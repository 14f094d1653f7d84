"""Sizes that the operators' C entries count in 32 bits: refused, never cut off to their low bits."""
import ctypes as C

import pytest


@pytest.mark.parametrize("V", [(1 << 31) - 4111, 1 << 31, 1 << 32, (1 << 32) + 5])
def test_linear_ce_refuses_more_items_than_it_counts(V):
    from recommenders.hip import load_library
    from recommenders.hip.linear_ce import V_MAX, _sizes
    with pytest.raises(ValueError, match="rows"):
        _sizes(4, V, 8)
    _sizes(4, V_MAX, 8)
    lib = load_library()
    assert lib.rg_linear_ce_work_floats(4, V_MAX, 8, 2) > 0
    assert lib.rg_linear_ce_work_floats(4, V_MAX + 1, 8, 2) == 0
    assert (1 << 32) + 5 != C.c_int((1 << 32) + 5).value   # what would have become of it on the way
