"""Sizes whose grids no launch takes (2^32 threads or more) are refused on the host, before anything is launched or allocated."""
import ctypes

import pytest

from paia_gemv.loader import KVCache

A = 1 << 20      # a 16-byte-aligned address, never dereferenced


def workspace(lib, kv_heads, B, T=1, group=4, width=8192):
    c = KVCache(A, A, 10, 16, kv_heads, 128)
    return lib._lib.paia_paged_attention_workspace(ctypes.byref(c), width, B, T, group * kv_heads)


@pytest.mark.parametrize("kv_heads,B,T", [(8, 2 ** 22, 1), (8, 2 ** 21, 1), (1, 2 ** 24, 1), (8, 2 ** 18, 64), (1, 2 ** 31 - 1, 1)])
def test_more_blocks_than_a_launch_takes(gemv_lib, kv_heads, B, T):
    for width in (0, 1, 8192):
        assert workspace(gemv_lib, kv_heads, B, T, width=width) == -2


@pytest.mark.parametrize("kv_heads,B,T", [(8, 2 ** 20, 1), (1, 2 ** 23, 1), (8, 2 ** 16, 64)])
def test_as_many_as_it_takes(gemv_lib, kv_heads, B, T):
    assert workspace(gemv_lib, kv_heads, B, T) > 0
