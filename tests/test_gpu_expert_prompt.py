"""The feed-forward half with experts over a prompt's tokens, all its operators together: every operator's output within a step
against its definition in 64 bits (tolerances as expert_util derives them), the step against the operators one by one, and a chunk of
a prompt replayed from a graph."""
import pytest
import torch

from decode_util import bits
from expert_util import experts64, order64, route64
from gpu_util import note
from paia_bench.expert_block import ExpertBlock
from paia_bench.timing import capture
from paia_gemv import ops
from test_gpu_expert_block import check_experts, check_norm, cpu

pytestmark = pytest.mark.gpu


def rows(tokens, hidden, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(tokens, hidden, generator=g).bfloat16().to(dev) for _ in range(2)]


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int4", "int4zp"])
@pytest.mark.parametrize("tokens,experts,chosen,absent", [(17, 8, 2, [3]), (61, 20, 4, []), (333, 6, 3, [0, 200, 332]), (1001, 40, 2, [])])
def test_a_prompt_and_its_parts(cuda, fmt, tokens, experts, chosen, absent):
    note(f"expert block, prompt {fmt} tokens {tokens} of {experts} take {chosen} absent {absent}")
    block = ExpertBlock(512, 384, experts, chosen, fmt, post_norm=tokens == 61, seed=tokens)
    y, r = rows(tokens, 512, tokens, cuda)
    gone = torch.zeros(tokens, dtype=torch.bool, device=cuda)
    gone[absent] = True
    out, residual = block.step(y, r, gone)

    x, r1 = ops.add_norm(y, r, block.norm, post_norm=block.post_norm)
    check_norm((x, r1), *cpu(y, r, block.norm), post_norm=None if block.post_norm is None else block.post_norm.cpu())
    logits = block.logits(x)
    all_of_them = torch.arange(tokens, dtype=torch.int32)
    want, bound = experts64("bf16", [block.router[None].cpu()], x.cpu(), all_of_them, torch.tensor([0, tokens]))
    assert ((logits.cpu().double() - want).abs() <= bound).all()
    ids, weights, order, offsets = block.route(x, gone)
    want_ids, want_w = route64(logits.masked_fill(gone[:, None], float("-inf")).cpu(), chosen)
    assert torch.equal(ids.cpu(), want_ids) and (ids.cpu()[absent] == -1).all()
    assert ((weights.cpu().double() - want_w).abs() <= (2.0 ** -24 + 2.0 ** -43) * want_w).all()
    assert all(torch.equal(a.cpu(), b) for a, b in zip((order, offsets), order64(want_ids, experts)))
    a = block.gate_up(x, order, offsets, gated=True)
    check_experts(block.gate_up, a, x, order, offsets, True)
    b = block.down(a, order, offsets)
    check_experts(block.down, b, a, order, offsets, False)
    parts = ops.add_norm(b.view(tokens, chosen, 512), r1, block.next_norm, weights=weights)
    check_norm(parts, *cpu(b.view(tokens, chosen, 512), r1, block.next_norm), weights=weights.cpu())
    assert torch.equal(bits(out), bits(parts[0])) and torch.equal(bits(residual), bits(parts[1]))
    assert torch.equal(bits(residual)[absent], bits(r1)[absent])      # a row without a token adds nothing


@pytest.mark.parametrize("fmt", ["fp8", "int4"])
def test_replays_of_a_chunk_follow_the_tokens(cuda, fmt):
    block = ExpertBlock(256, 256, 12, 3, fmt, seed=1)
    y, r = rows(90, 256, 2, cuda)
    gone, out = torch.zeros(90, dtype=torch.bool, device=cuda), {}
    graph = capture(lambda: out.update(step=block.step(y, r, gone)))
    for i, absent in enumerate(([], [0, 8], list(range(90)), list(range(40, 90)))):
        y.copy_(rows(90, 256, 10 + i, cuda)[0])
        gone.zero_()
        gone[absent] = True
        junk = torch.randn(1 << 18, device=cuda).mul_(2.0)
        torch.cuda.synchronize()
        note(f"expert block, replay of a chunk {fmt} {i}")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out["step"], block.step(y, r, gone)))
        del junk
