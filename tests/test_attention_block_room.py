"""AttentionBlock past the room of its sequences: the block table is not read beyond its width, nothing is written."""
import pytest
import torch

from paia_bench.attention_block import AttentionBlock


def test_slots_past_the_room():
    block = AttentionBlock.__new__(AttentionBlock)
    block.page_size, block.table = 16, torch.tensor([[5, 2, -1], [7, -1, -1]], dtype=torch.int32)
    for at, want in ((0, [80, 112]), (15, [95, 127]), (16, [32, None]), (31, [47, None]), (32, [None] * 2), (48, [None] * 2),
                     (10 ** 9, [None] * 2)):
        block.positions = torch.tensor([at, at])
        got = block.slots().tolist()
        assert all(g < 0 if w is None else g == w for g, w in zip(got, want)), (at, got)


@pytest.mark.gpu
def test_steps_past_the_room(cuda):
    from decode_util import bits
    from gpu_util import note
    block = AttentionBlock("qwen25_7b", "bf16", [17, 3], room=2, cache="bf16")
    assert block.table.shape == (2, 3) and block.table[:, -1].tolist() == [-1, -1]
    x = torch.randn(2, block.qkv.K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    for i in range(15):
        note(f"attention block room step {i}")
        y = block.step(x)
    assert block.positions.tolist() == [32, 18] and y[0].isfinite().all()
    k, v = block.k_cache.clone(), block.v_cache.clone()
    for i in range(40):
        note(f"attention block past the room step {i}")
        block.step(x)
    torch.cuda.synchronize()
    assert torch.equal(bits(block.k_cache), bits(k)) and torch.equal(bits(block.v_cache), bits(v))
