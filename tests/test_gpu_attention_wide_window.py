"""Windows as wide as 32 bits hold, on tables as wide, with more tokens than positions: they hide nothing."""
import pytest
import torch

from decode_util import bits
from gpu_util import note
from paia_gemv import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,T", [(100, 8192), (5000, 8192), (3, 1)])
def test_windows_that_hide_nothing(cuda, n, T):
    g = torch.Generator(device=cuda).manual_seed(n)
    k, v = (torch.randn(1, 1, 2 ** 20, 64, dtype=torch.bfloat16, device=cuda, generator=g) for _ in range(2))
    q = torch.randn(1, T, 1, 64, dtype=torch.bfloat16, device=cuda, generator=g)
    table = torch.zeros(1, 2 ** 11 + 1, dtype=torch.int32, device=cuda)          # 2^31 positions and more, on one page
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    want, wlse = ops.paged_attention(q, k, v, table, lens, return_lse=True)
    first = max(0, T - n)                       # the first token that sees a position
    assert want[0, :first].eq(0).all() and wlse[0, :first].isneginf().all() and wlse[0, first:].isfinite().all()
    for window in (2 ** 31 - 1, 2 ** 31 - 5000, n):
        note(f"attention window={window} n={n} T={T}")
        out, lse = ops.paged_attention(q, k, v, table, lens, window=window, return_lse=True)
        assert torch.equal(bits(out), bits(want)) and torch.equal(lse, wlse), window
