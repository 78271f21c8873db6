"""rope_append on more tokens than one launch takes (a launch has less than 2^32 threads, here 64 a token)."""
import pytest
import torch

from decode_util import bits
from gpu_util import note
from paia_gemv import ops

pytestmark = pytest.mark.gpu


def test_tokens_beyond_a_launch(cuda):
    """2^26 + 5 tokens of one query and one key head, all of the same row at seven positions in turn, a few of them with a slot. q
    and the cache equal the small calls bit for bit."""
    M, period = 2 ** 26 + 5, 7
    g = torch.Generator().manual_seed(3)
    table = ops.rope_table(32, 64, device=cuda)
    row = torch.randn(1, 192, generator=g).to(torch.bfloat16).to(cuda)
    qkv = row.expand(M, 192)                                     # stride 0: 26 GB otherwise
    positions = torch.arange(M, device=cuda) % period
    slots = torch.full((M,), -1, dtype=torch.int64, device=cuda)
    kept = [0, 5, 2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1, 2 ** 26 - 1, 2 ** 26, M - 1]
    slots[torch.tensor(kept, device=cuda)] = torch.arange(len(kept), device=cuda)
    k, v = (torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    want = ops.rope_append(row.expand(period, 192).contiguous(), positions[:period], table, k.clone(), v.clone(),
                           torch.full((period,), -1, dtype=torch.int64, device=cuda), 1)
    note(f"rope M={M}")
    q = ops.rope_append(qkv, positions, table, k, v, slots, 1)
    torch.cuda.synchronize()
    whole = M // period * period
    per = 1 << 20
    for at in range(0, whole, per * period):
        part = q[at:min(at + per * period, whole)].view(-1, period, 64)
        assert (part.view(torch.int16) == want.view(1, period, 64).view(torch.int16)).all(), at
    assert torch.equal(bits(q[whole:]), bits(want[:M - whole]))
    small_k, small_v = torch.zeros_like(k), torch.zeros_like(v)
    ops.rope_append(row.expand(len(kept), 192).contiguous(), positions[torch.tensor(kept, device=cuda)], table, small_k, small_v,
                    torch.arange(len(kept), device=cuda), 1)
    assert torch.equal(bits(k), bits(small_k)) and torch.equal(bits(v), bits(small_v)) and k[0, 0, :len(kept)].ne(0).any()
