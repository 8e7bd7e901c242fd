"""Query heads that share a KV head: the C entry points take up to 32, as the Python side does, which is what the kernels' division
by their number holds for.  Nothing here reaches a GPU: calls with too many are refused, and the others only sized."""

import ctypes

import pytest

from flashbob_b200 import _lib
from test_cabi_paged import FAKE, _paged


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,max_pages", [(1, 64), (2, 64), (300, 64), (3, 1 << 20)])
def test_larger_groups_are_refused(bits, N, max_pages):
    lib = _lib.load()
    for heads, group in ((8, 32), (1, 32), (1, 1)):
        assert lib.bob_sm100_paged_workspace_bytes(ctypes.byref(_paged(N=N, Hq=heads * group, heads=heads, bits=bits, max_pages=max_pages))) >= 256
    for heads, group in ((8, 33), (1, 33), (1, 64), (1, 257), (2, 4096)):
        a = _paged(N=N, Hq=heads * group, heads=heads, bits=bits, max_pages=max_pages)
        assert lib.bob_sm100_paged_workspace_bytes(ctypes.byref(a)) == 0
        assert lib.bob_sm100_paged_fwd(ctypes.byref(a), FAKE, None) == -2


def test_the_kernels_division_of_rows_by_the_group():
    """Row r of an item is a head of token (r + skip) / G, r below 32 and skip below G, computed as x (65536 / G + 1) / 65536."""
    for G in range(1, 33):
        assert all(x * (65536 // G + 1) >> 16 == x // G for x in range(64))
    assert 256 * (65536 // 257 + 1) >> 16 == 1                   # what went wrong from 257 on
