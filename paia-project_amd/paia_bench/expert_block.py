"""The feed-forward half of a decode layer with experts on one GPU, every operator of it from this library:

    attention's output y, residual r -> norm behind the attention (optional), residual and norm -> router logits -> each token's
    experts -> their gate and up projections (silu(gate) * up) -> their down projections -> sum by the router's weights,
    residual and the next layer's norm

for a batch of tokens, one of each sequence, or a prompt's. Rows without a token (a captured batch that is not full) are marked in
`absent`: they choose no experts. Weights are random (seeded), every expert of the size of the model's feed-forward block.

    python -m paia_bench.expert_block --model llama31_8b --fmt fp8 --experts 8 --chosen 2 --batch 8

times a step of a decode batch. The layer's experts together can exceed the 256 MiB last-level cache by far while the chosen ones lie in it whole, so
the command steps as many blocks in turn (`copies`) as keep any of them from being found there when it is next used.
"""
from __future__ import annotations

import argparse
import json
import sys

import torch

from paia_gemv import ops, quant
from paia_gemv.shapes import LAYER

from .timing import capture, plan_rotation, replay_ms, stats


class Experts:
    """`experts` matrices [N, K] in one of the library's formats."""

    def __init__(self, fmt, experts, N, K, gen):
        self.fmt = fmt
        W = lambda: torch.randn(N, K, generator=gen, device=gen.device) * K ** -0.5  # noqa: E731
        if fmt == "bf16":
            made = [(W().to(torch.bfloat16),) for _ in range(experts)]
        elif fmt in ("fp8", "int4", "int4zp"):
            q = {"fp8": quant.quantize_fp8_rowwise, "int4": quant.quantize_int4_g128, "int4zp": quant.quantize_int4_zp_g128}[fmt]
            made = [q(W()) for _ in range(experts)]
        else:
            raise ValueError(f"unknown weight format {fmt!r}")
        self.w = tuple(torch.stack(parts) for parts in zip(*made))

    def __call__(self, x, order, offsets, gated=False):
        call = {"bf16": ops.experts_bf16, "fp8": ops.experts_fp8, "int4": ops.experts_int4, "int4zp": ops.experts_int4_zp}
        return call[self.fmt](*self.w, x, order, offsets, gated=gated)

    def bytes(self):
        """Of one expert."""
        return sum(t[0].numel() * t.element_size() for t in self.w)


class ExpertBlock:
    """Weights of one layer: `experts` experts of `ffn` hidden values, `chosen` a token, router in bf16, norms around the block."""

    def __init__(self, hidden, ffn, experts, chosen, fmt, post_norm=False, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        bf16 = lambda *s, by=1.0: (torch.randn(*s, generator=gen, device=device) * by).to(torch.bfloat16)  # noqa: E731
        self.hidden, self.chosen = hidden, chosen
        self.router = bf16(experts, hidden, by=hidden ** -0.5)
        self.gate_up = Experts(fmt, experts, 2 * ffn, hidden, gen)
        self.down = Experts(fmt, experts, hidden, ffn, gen)
        self.norm, self.next_norm = bf16(hidden, by=0.1) + 1.0, bf16(hidden, by=0.1) + 1.0
        self.post_norm = bf16(hidden, by=0.1) + 1.0 if post_norm else None

    def logits(self, x):
        """The router's product with x [tokens, hidden], bf16 [tokens, experts]: up to 16 rows as a small batch, more as the product
        with the one expert that all of them have chosen."""
        tokens = len(x)
        if tokens <= 16:
            return ops.gemv_bf16(self.router, x)
        order = torch.arange(tokens, dtype=torch.int32, device=x.device)
        offsets = torch.arange(0, tokens + 1, tokens, dtype=torch.int32, device=x.device)
        return ops.experts_bf16(self.router[None], x, order, offsets)

    def route(self, x, absent=None):
        logits = self.logits(x)
        if absent is not None:
            logits = logits.masked_fill(absent[:, None], float("-inf"))
        return ops.route_experts(logits, self.chosen)

    def step(self, y, residual, absent=None):
        """y, residual bf16 [tokens, hidden] -> (x of the next layer, residual), bf16 [tokens, hidden]."""
        x, residual = ops.add_norm(y, residual, self.norm, post_norm=self.post_norm)
        _, weights, order, offsets = self.route(x, absent)
        a = self.gate_up(x, order, offsets, gated=True)
        a = self.down(a, order, offsets)
        return ops.add_norm(a.view(len(x), self.chosen, self.hidden), residual, self.next_norm, weights=weights)

    def bytes(self, used):
        """Bytes of weights that a step over `used` different experts cannot do without."""
        return self.router.numel() * 2 + used * (self.gate_up.bytes() + self.down.bytes())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--model", choices=sorted(LAYER), default="llama31_8b")
    ap.add_argument("--fmt", choices=("bf16", "fp8", "int4", "int4zp"), default="fp8")
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--chosen", type=int, default=2)
    ap.add_argument("--ffn", type=int, default=0, help="hidden values of an expert; 0: the model's")
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args(argv)
    if not 1 <= a.batch <= 16:
        ap.error("--batch: 1 to 16 sequences")
    if not 1 <= a.chosen <= a.experts:
        ap.error("--chosen: 1 to --experts")
    _, hidden, down = next(shape for shape in LAYER[a.model] if shape[0] == "down")
    make = lambda seed: ExpertBlock(hidden, a.ffn or down, a.experts, a.chosen, a.fmt, seed=seed)  # noqa: E731
    blocks = [make(0)]
    y, r = (torch.randn(a.batch, hidden, device="cuda").to(torch.bfloat16) for _ in range(2))
    used = lambda block: len(set(block.route(ops.add_norm(y, r, block.norm)[0])[0].flatten().tolist()))  # noqa: E731
    plan = plan_rotation(blocks[0].bytes(used(blocks[0])))
    blocks += [make(seed) for seed in range(1, plan["n_copies"])]
    nbytes = sum(block.bytes(used(block)) for block in blocks)
    graph = capture(lambda: [block.step(y, r) for block in blocks], warm=2)
    us = stats(replay_ms(graph, a.steps))["median"] * 1e3
    print(json.dumps({"model": a.model, "fmt": a.fmt, "experts": a.experts, "chosen": a.chosen, "ffn": a.ffn or down,
                      "batch": a.batch, "copies": len(blocks), "llc_safe": plan["llc_safe"],
                      "us_per_step": round(us / len(blocks), 2), "gbps": round(nbytes / us / 1e3, 1)}))
    return 0


if __name__ == "__main__":
    sys.exit(main())
