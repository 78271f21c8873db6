"""The feed-forward half of a decode layer with experts, all its operators together: every operator's output within a step against
its definition in 64 bits (tolerances as expert_util derives them), the step against the operators one by one, replayed graphs
against eager steps, and both halves of a layer in one graph."""
import json

import pytest
import torch

from decode_util import BF16_HALF, bits
from expert_util import experts64, norm64, order64, route64
from gpu_util import note
from paia_bench.attention_block import AttentionBlock
from paia_bench.expert_block import ExpertBlock, main
from paia_bench.timing import LLC_BYTES, capture
from paia_gemv import ops

pytestmark = pytest.mark.gpu


def cpu(*tensors):
    return [t.detach().cpu() for t in tensors]


def check_norm(got, x, residual, norm, **more):
    h, r, eh, er = norm64(x, residual, norm, **more)
    for out, want, err in ((got[0], h, eh), (got[1], r, er)):
        assert ((out.cpu().double() - want).abs() <= err + BF16_HALF * (want.abs() + err)).all()


def check_experts(experts, out, x, order, offsets, gated):
    W = [w.cpu() for w in experts.w]
    if experts.fmt == "fp8":
        W[0] = W[0].view(torch.float8_e4m3fn)
    want, bound = experts64(experts.fmt, W, x.cpu(), order.cpu(), offsets.cpu(), None, gated)
    assert ((out.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int4", "int4zp"])
@pytest.mark.parametrize("tokens,experts,chosen,absent", [(1, 8, 2, []), (5, 6, 3, [1, 4]), (16, 20, 4, [15]), (3, 4, 4, [0, 1, 2])])
def test_a_step_and_its_parts(cuda, fmt, tokens, experts, chosen, absent):
    note(f"expert block {fmt} tokens {tokens} of {experts} take {chosen} absent {absent}")
    block = ExpertBlock(512, 384, experts, chosen, fmt, post_norm=tokens == 5, seed=tokens)
    g = torch.Generator().manual_seed(tokens)
    y, r = (torch.randn(tokens, 512, generator=g).bfloat16().to(cuda) for _ in range(2))
    gone = torch.zeros(tokens, dtype=torch.bool, device=cuda)
    gone[absent] = True
    out, residual = block.step(y, r, gone)

    x, r1 = ops.add_norm(y, r, block.norm, post_norm=block.post_norm)
    check_norm((x, r1), *cpu(y, r, block.norm), post_norm=None if block.post_norm is None else block.post_norm.cpu())
    ids, weights, order, offsets = block.route(x, gone)
    logits = ops.gemv_bf16(block.router, x).masked_fill(gone[:, None], float("-inf"))
    want_ids, want_w = route64(logits.cpu(), chosen)
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


@pytest.mark.parametrize("fmt", ["fp8", "int4zp"])
def test_replays_follow_the_tokens(cuda, fmt):
    block = ExpertBlock(256, 256, 12, 3, fmt, seed=1)
    g = torch.Generator().manual_seed(2)
    y, r = (torch.randn(9, 256, generator=g).bfloat16().to(cuda) for _ in range(2))
    gone, out = torch.zeros(9, dtype=torch.bool, device=cuda), {}
    graph = capture(lambda: out.update(step=block.step(y, r, gone)))
    for i, absent in enumerate(([], [0, 8], list(range(9)), [3])):
        y.copy_(torch.randn(9, 256, generator=g).bfloat16())
        gone.zero_()
        gone[absent] = True
        junk = torch.randn(1 << 18, device=cuda).mul_(2.0)
        torch.cuda.synchronize()
        note(f"expert block replay {fmt} {i}")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out["step"], block.step(y, r, gone)))
        del junk


def test_both_halves_of_a_layer(cuda):
    """Attention, then experts, token after token in one graph, as eager steps of a twin."""
    note("attention and experts")

    def make():
        return (AttentionBlock("qwen25_7b", "fp8", [40, 3, 17], room=20, cache="fp8", seed=3),
                ExpertBlock(3584, 256, 8, 2, "int4", post_norm=True, seed=4))

    def layer(halves, x, r):
        attention, experts = halves
        return experts.step(attention.step(x), r)

    g = torch.Generator().manual_seed(5)
    x, r = (torch.randn(3, 3584, generator=g).bfloat16().to(cuda) for _ in range(2))
    halves, twin, out = make(), make(), {}
    graph = capture(lambda: out.update(y=layer(halves, x, r)), warm=1)
    layer(twin, x, r)
    for i in range(3):
        want = layer(twin, x, r)
        note(f"attention and experts, replay {i}")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(out["y"], want))
        assert want[0].isfinite().all()


def test_command(cuda, capsys):
    note("expert block command")
    assert main(["--model", "qwen25_7b", "--fmt", "int4zp", "--experts", "16", "--chosen", "4", "--ffn", "2560", "--batch", "3",
                 "--steps", "4"]) == 0
    r = json.loads(capsys.readouterr().out.splitlines()[-1])
    one = 3 * 2560 * 3584 // 2                               # codes alone of the smallest share: four experts
    assert r["us_per_step"] > 0 and r["llc_safe"] is True and r["copies"] * 4 * one <= 64 * 2 ** 30
    assert r["gbps"] < 8000 and r["copies"] * 12 * (one + 3 * 2560 * 28 * 3 + 2 ** 20) >= 4 * LLC_BYTES
    for bad in (["--batch", "17"], ["--chosen", "9"], ["--chosen", "0"]):
        with pytest.raises(SystemExit):
            main(bad)


@pytest.mark.parametrize("fmt", ["bf16", "int4"])
def test_two_steps_at_once(cuda, fmt):
    """Steps of two sizes on two streams, over and over, each as alone."""
    block = ExpertBlock(1024, 512, 16, 4, fmt, seed=6)
    g = torch.Generator().manual_seed(7)
    sizes = (2, 16)
    rows = [[torch.randn(n, 1024, generator=g).bfloat16().to(cuda) for _ in range(2)] for n in sizes]
    want = [[t.clone() for t in block.step(*r)] for r in rows]
    streams = [torch.cuda.Stream() for _ in sizes]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    note(f"expert block on two streams {fmt}")
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(block.step(*rows[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(bits(a), bits(b)) for step in got[i] for a, b in zip(step, want[i]))


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int4", "int4zp"])
def test_the_same_expert_twice(cuda, fmt):
    """Ids that name an expert more than once, or one that is not there: pairs of their own, and zeros."""
    block = ExpertBlock(2048, 128, 6, 3, fmt, seed=8)
    ids = torch.tensor([[4, 4, 4], [1, 9, 1], [-1, -1, -1], [0, 5, 4]], dtype=torch.int32, device=cuda)
    x = torch.randn(4, 2048, generator=torch.Generator().manual_seed(9)).bfloat16().to(cuda)
    note(f"the same expert twice {fmt}")
    order, offsets = ops.expert_order(ids, 6)
    out = block.gate_up(x, order, offsets, gated=True).view(4, 3, -1)
    check_experts(block.gate_up, out.view(12, -1), x, order, offsets, True)
    assert torch.equal(bits(out[0, 0]), bits(out[0, 1])) and torch.equal(bits(out[0, 0]), bits(out[0, 2]))
    assert torch.equal(bits(out[1, 0]), bits(out[1, 2])) and not bits(out[1, 1]).any() and not bits(out[2]).any()
