"""What the attention block's command prints: a rate that is not the last-level cache's, over the bytes of the timed steps."""
import json

import pytest
import torch

from paia_bench.attention_block import AttentionBlock, main
from paia_bench.timing import LLC_BYTES
from paia_gemv.shapes import gemv_bytes


def test_bytes_follow_the_positions():
    block = AttentionBlock.__new__(AttentionBlock)

    class Weights:
        @staticmethod
        def bytes(M):
            return 1000 * M
    block.heads, block.qkv, block.o = (32, 8, 128), Weights, Weights
    block.positions, block.k_cache = torch.tensor([10, 0, 5]), torch.empty(1, dtype=torch.bfloat16)
    row = 2 * 8 * 128 * 2
    assert block.bytes() == 6000 + (15 + 3) * row            # each new token's own position included
    assert block.bytes(7) == 6000 + (15 + 3 * 8) * row


@pytest.mark.gpu
def test_the_command_leaves_the_last_level_cache(cuda, capsys):
    from gpu_util import note
    note("attention block command, rotation")
    assert main(["--model", "llama31_8b", "--fmt", "int4zp", "--batch", "2", "--context", "100", "--steps", "4"]) == 0
    r = json.loads(capsys.readouterr().out.splitlines()[-1])
    weights = sum(gemv_bytes("int4zp", N, 4096, False, 2)["total"] for N in (6144, 4096))
    cache = 2 * 8 * 128 * 2 * (100 + 50 + 2 * (2 + 4 // 2 + 1))
    assert r["llc_safe"] is True and r["copies"] * (weights + cache) >= 4 * LLC_BYTES
    assert abs(r["gbps"] - (weights + cache) / r["us_per_step"] / 1e3) <= 0.01 * r["gbps"] and r["gbps"] < 8000
