"""The attention half of a decode layer, all its operators together: eager steps and a replayed graph, against the same chain
from the definitions in 64 bits (rounded to bf16 where the operators store bf16).

Gate: max |y - ref| / max |ref| < 2e-2, the gate of this suite's other end-to-end comparisons.
"""
import pytest
import torch

from decode_util import attention64, bits, codes, lora64, on, rope64
from gpu_util import note
from paia_bench.attention_block import AttentionBlock
from paia_bench.timing import capture

pytestmark = pytest.mark.gpu
GATE = 2e-2


def project64(p, x, ids):
    y = x.double() @ p.weights().cpu().double().t()
    if p.bias is not None:
        y = y + p.bias.cpu().double()
    y = y.to(torch.bfloat16)
    if p.A is not None:
        y = lora64(y, x, p.A.cpu(), p.B.cpu(), ids, p.scaling.cpu(), p.splits).to(torch.bfloat16)
    return y


def step64(block, x):
    """One step from the block's present state (which it leaves alone): y, and the cache with the new rows."""
    heads, kv_heads, dim = block.heads
    ids, pos, table = block.ids.cpu(), block.positions.cpu(), block.table.cpu()
    qkv = project64(block.qkv, x, ids)
    q, k, v = rope64(qkv, pos, block.cos_sin.cpu(), heads, kv_heads, dim)
    caches, scales = [], [block.k_scale, block.v_scale]
    for cache, rows, s in ((block.k_cache, k, scales[0]), (block.v_cache, v, scales[1])):
        c = on(cache.detach(), "cpu").clone()
        if s is not None:
            rows = (rows / s.cpu().double()[:, None]).clamp(-448, 448).float()
        for b in range(len(pos)):
            p = int(pos[b])
            c[int(table[b, p // block.page_size]), :, p % block.page_size] = rows[b].to(c.dtype)
        caches.append(c)
    cpu = [None if s is None else s.cpu() for s in scales]
    a = attention64(q[:, None].to(torch.bfloat16), *caches, table, pos + 1, k_scale=cpu[0], v_scale=cpu[1])[0]
    return project64(block.o, a.view(len(pos), -1).to(torch.bfloat16), ids), caches


def gate(y, ref):
    rel = float((y.cpu().double() - ref.double()).abs().max() / ref.double().abs().max())
    assert rel < GATE, rel


@pytest.mark.parametrize("model,fmt,cache,lengths,adapters", [
    ("llama31_8b", "fp8", "bf16", [300], 0),
    ("llama31_8b", "int4zp", "fp8", [1, 700, 33, 0], 2),
    ("qwen25_7b", "bf16", "fp8", [129, 64], 1),
    ("qwen25_7b", "int4", "bf16", [40, 15, 16, 17, 250], 3),
])
def test_steps(cuda, model, fmt, cache, lengths, adapters):
    note(f"attention block {model} {fmt} cache {cache} lengths {lengths} adapters {adapters}")
    block = AttentionBlock(model, fmt, lengths, room=20, cache=cache, adapters=adapters, seed=3)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(len(lengths), block.qkv.K, generator=g).to(torch.bfloat16)
    for _ in range(2):
        ref, caches = step64(block, x)
        y = block.step(x.to(cuda))
        torch.cuda.synchronize()
        gate(y, ref)
        for got, want in zip((block.k_cache, block.v_cache), caches):
            a, b = codes(got), codes(want)
            assert float((a - b).abs().max() / b.abs().max()) < GATE
    # a captured step goes on from there, token after token, as eager steps of a twin do
    twin = AttentionBlock(model, fmt, lengths, room=20, cache=cache, adapters=adapters, seed=3)
    xd, out = x.to(cuda), {}
    graph = capture(lambda: out.update(y=block.step(xd)), warm=1)       # one eager step more
    for _ in range(3):
        twin.step(xd)
    for i in range(4):
        want = twin.step(xd)
        junk = torch.randn(1 << 18, device=cuda).mul_(2.0)
        torch.cuda.synchronize()
        note(f"attention block replay {i}")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(block.positions, twin.positions)
        assert torch.equal(bits(out["y"]), bits(want)), i
        assert torch.equal(bits(block.k_cache), bits(twin.k_cache)) and torch.equal(bits(block.v_cache), bits(twin.v_cache))
        del junk


def test_command(cuda, capsys):
    import json

    from paia_bench.attention_block import main
    note("attention block command")
    assert main(["--model", "qwen25_7b", "--fmt", "int4zp", "--batch", "3", "--context", "200", "--adapters", "2",
                 "--steps", "4"]) == 0
    assert json.loads(capsys.readouterr().out.splitlines()[-1])["us_per_step"] > 0
    with pytest.raises(SystemExit):
        main(["--batch", "17"])
