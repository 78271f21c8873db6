"""paged_attention_workspace where there are shapes alone, so that what sizes a workspace with it can be traced: the figure is the
C ABI's, and refusals stay refusals."""
import ctypes

import pytest
import torch

from paia_gemv import ops
from paia_gemv.loader import KVCache


def wanted(lib, fp8, width, B, T, heads):
    c = KVCache(1 << 20, 1 << 20, 10, 16, 8, 128, fp8)
    return lib._lib.paia_paged_attention_workspace(ctypes.byref(c), width, B, T, heads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.uint8])
@pytest.mark.parametrize("width,B,T,heads", [(1000, 2, 1, 32), (1, 3, 1, 8), (8192, 16, 5, 64)])
def test_meta(gemv_lib, dtype, width, B, T, heads):
    cache = torch.empty(10, 8, 16, 128, dtype=dtype, device="meta")
    need = ops.paged_attention_workspace(cache, width, B, T, heads)
    assert need == wanted(gemv_lib, dtype != torch.bfloat16, width, B, T, heads)
    assert ops.paged_attention_workspace(cache.transpose(1, 2).contiguous().transpose(1, 2), width, B, T, heads) == need


def test_meta_refusals(gemv_lib):
    cache = torch.empty(10, 8, 16, 128, dtype=torch.bfloat16, device="meta")
    for a in ((cache, 1000, 2, 1, 30), (cache, -1, 2, 1, 32), (cache[..., :96], 1000, 2, 1, 32)):
        with pytest.raises(RuntimeError, match="-2"):
            ops.paged_attention_workspace(*a)
    for bad in (cache.half(), cache[0], cache[:0], cache.transpose(2, 3)):
        with pytest.raises(RuntimeError, match="cache"):
            ops.paged_attention_workspace(bad, 1000, 2, 1, 32)


def test_fake_tensors(gemv_lib):
    """A function that sizes its workspace and attends, traced on fake tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops.load()
    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
        cache = e(10, 8, 16, 128)
        need = ops.paged_attention_workspace(cache, 1000, 2, 1, 32)
        space = torch.empty(need, dtype=torch.uint8, device="meta")
        out = ops.paged_attention(e(2, 32, 128), cache, cache, e(2, 1000, dtype=torch.int32), e(2, dtype=torch.int32),
                                  workspace=space)
        assert out.shape == (2, 32, 128)
    assert need == wanted(gemv_lib, False, 1000, 2, 1, 32) > 0
