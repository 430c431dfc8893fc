"""CPU tests of the cache operators' refusals at the edges of what their header allows (no device
needed: every refusal here happens before the library touches one)."""
import ctypes as C

import pytest

from test_cache_ops_cpu import INVALID, P, tree


@pytest.mark.parametrize("stride,cols", [(64, 0), (64, -1), (64, 65), (0, 0)])
def test_rows_of_weights_hold_their_columns(ckl, stride, cols):
    L = ckl.lib()
    assert L.ckl_cache_weights_ex(C.byref(tree(ckl)), P, P, stride, cols, 1.0, None) == INVALID
    assert L.ckl_cache_select_ex(P, stride, cols, P, P, 2, 8, 0, 0, P, P, None) == INVALID
    assert L.ckl_cache_compact_ex(P, 0x100000, P, P, P, 2, 2, 4, P, 8, P, None, P, stride, cols, None,
                                  None) == INVALID
