"""The attention half of a decode layer on one GPU, every operator of it from this library:

    x -> qkv projection (+ adapters) -> head rotation and cache write -> attention over the paged cache -> o projection
    (+ adapters) -> y

for a batch of sequences of their own lengths, each row with an adapter of its own or none. One `step` is one token of every
sequence; it advances the positions on the device, so a captured step is replayed token after token. Weights, cache contents
and adapters are random (seeded); Qwen2.5's qkv projection has its bias.

    python -m paia_bench.attention_block --model llama31_8b --fmt fp8 --cache fp8 --batch 8 --context 4096 --adapters 4

times a step. One layer's weights and cache can lie in the 256 MiB last-level cache whole, so the command steps as many blocks in
turn (`copies`) as keep any of them from being found there when it is next used.
"""
from __future__ import annotations

import argparse
import json
import sys

import torch

from paia_gemv import ops, quant
from paia_gemv.shapes import HEADS, LAYER, ROPE_BASE, gemv_bytes

from .timing import capture, plan_rotation, replay_ms, stats


class Projection:
    """One weight matrix [N, K] in one of the library's formats, and low-rank adapters beside it."""

    def __init__(self, fmt, N, K, bias, splits, adapters, rank, gen):
        dev = gen.device
        self.fmt, self.N, self.K, self.splits = fmt, N, K, splits
        W = torch.randn(N, K, generator=gen, device=dev) * 0.02
        if fmt == "bf16":
            self.w = (W.to(torch.bfloat16),)
        elif fmt == "fp8":
            self.w = quant.quantize_fp8_rowwise(W)
        elif fmt == "int4":
            self.w = quant.quantize_int4_g128(W)
        elif fmt == "int4zp":
            self.w = quant.quantize_int4_zp_g128(W)
        else:
            raise ValueError(f"unknown weight format {fmt!r}")
        self.bias = (torch.randn(N, generator=gen, device=dev) * 0.02).to(torch.bfloat16) if bias else None
        self.A = self.B = self.scaling = None
        if adapters:
            S = len(splits)
            self.A = (torch.randn(adapters, S * rank, K, generator=gen, device=dev) * K ** -0.5).to(torch.bfloat16)
            self.B = (torch.randn(adapters, N, rank, generator=gen, device=dev) * 0.3 * rank ** -0.5).to(torch.bfloat16)
            self.scaling = torch.rand(adapters, generator=gen, device=dev) + 0.5

    def weights(self):
        """The matrix that the format stands for, fp32 [N, K]."""
        if self.fmt == "bf16":
            return self.w[0].float()
        return {"fp8": quant.dequant_fp8, "int4": quant.dequant_int4, "int4zp": quant.dequant_int4_zp}[self.fmt](*self.w)

    def __call__(self, x, ids):
        if self.fmt == "int4":
            y = ops.gemv_int4(*self.w, x)
            if self.bias is not None:
                y += self.bias
        else:
            y = {"bf16": ops.gemv_bf16, "fp8": ops.gemv_fp8, "int4zp": ops.gemv_int4_zp}[self.fmt](*self.w, x,
                                                                                               bias=self.bias)
        if self.A is not None:
            ops.lora_add(y, x, self.A, self.B, ids, scaling=self.scaling, splits=self.splits, out=y)
        return y

    def bytes(self, M):
        return gemv_bytes(self.fmt, self.N, self.K, self.bias is not None, M)["total"]


class AttentionBlock:
    """Weights, paged cache and bookkeeping of `batch` sequences with `lengths` positions in the cache and room for `room`
    more. cache "bf16" or "fp8"."""

    def __init__(self, model, fmt, lengths, room=64, cache="bf16", page_size=16, adapters=0, rank=16, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.model, self.heads = model, HEADS[model]
        heads, kv_heads, dim = self.heads
        (_, Nq, Kq), (_, No, Ko) = LAYER[model][:2]
        self.qkv = Projection(fmt, Nq, Kq, model.startswith("qwen"), [heads * dim, kv_heads * dim, kv_heads * dim],
                              adapters, rank, gen)
        self.o = Projection(fmt, No, Ko, False, [No], adapters, rank, gen)
        B = len(lengths)
        need = [-(-(n + room) // page_size) for n in lengths]
        self.page_size, width = page_size, max(need)
        order = torch.randperm(sum(need), generator=gen, device=device).int()
        # a column more than any sequence has pages, for positions past the room: page -1, nothing is written or attended there
        self.table = torch.full((B, width + 1), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (sum(need), kv_heads, page_size, dim)
        self.k_scale = self.v_scale = None
        if cache == "fp8":
            draw = lambda: (torch.randn(shape, generator=gen, device=device) * 20).to(torch.float8_e4m3fn)  # noqa: E731
            self.k_scale, self.v_scale = (torch.full((kv_heads,), 0.05, device=device) for _ in range(2))
        elif cache == "bf16":
            draw = lambda: torch.randn(shape, generator=gen, device=device, dtype=torch.bfloat16)  # noqa: E731
        else:
            raise ValueError(f"unknown cache type {cache!r}")
        self.k_cache, self.v_cache = draw(), draw()
        self.positions = torch.tensor(lengths, dtype=torch.int64, device=device)    # of the next token
        self.cos_sin = ops.rope_table(width * page_size, dim, ROPE_BASE[model], device=device)
        self.ids = (torch.arange(B, device=device) % (adapters + 1) - 1).int()      # row 0 without an adapter
        self.workspace = torch.empty(max(16, ops.paged_attention_workspace(self.k_cache, width + 1, B, 1, heads)),
                                     dtype=torch.uint8, device=device)

    def slots(self):
        """Where the next token of every sequence goes, negative past its room."""
        column = (self.positions // self.page_size).clamp(max=self.table.shape[1] - 1)
        return self.table.gather(1, column[:, None])[:, 0].long() * self.page_size + self.positions % self.page_size

    def step(self, x):
        """x bf16 [batch, hidden] -> y bf16 [batch, hidden]: the next token of every sequence. Past its room a sequence's cache stays
        as it is."""
        heads, _, dim = self.heads
        slots = self.slots()
        lens = (self.positions + 1).int()
        qkv = self.qkv(x, self.ids)
        q = ops.rope_append(qkv, self.positions, self.cos_sin, self.k_cache, self.v_cache, slots, heads,
                            k_scale=self.k_scale, v_scale=self.v_scale)
        a = ops.paged_attention(q, self.k_cache, self.v_cache, self.table, lens, k_scale=self.k_scale, v_scale=self.v_scale,
                                workspace=self.workspace)
        y = self.o(a.view(len(x), heads * dim), self.ids)
        self.positions += 1
        return y

    def bytes(self, later=0):
        """Bytes that the step after `later` more cannot do without: weights, activations and the cache as it stands then (adapters
        left out)."""
        _, kv_heads, dim = self.heads
        M = len(self.positions)
        return (self.qkv.bytes(M) + self.o.bytes(M)
                + int(self.positions.sum() + M * (later + 1)) * 2 * kv_heads * dim * self.k_cache.element_size())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--model", choices=sorted(HEADS), default="llama31_8b")
    ap.add_argument("--fmt", choices=("bf16", "fp8", "int4", "int4zp"), default="fp8")
    ap.add_argument("--cache", choices=("bf16", "fp8"), default="bf16")
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--context", type=int, default=4096, help="positions of the longest sequence; the others are shorter")
    ap.add_argument("--adapters", type=int, default=0)
    ap.add_argument("--rank", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args(argv)
    if not 1 <= a.batch <= 16:
        ap.error("--batch: the projections take 1 to 16 rows")
    lengths = [max(1, a.context * (a.batch - b) // a.batch) for b in range(a.batch)]
    make = lambda seed: AttentionBlock(a.model, a.fmt, lengths, room=a.steps + 16, cache=a.cache, adapters=a.adapters,  # noqa: E731
                                       rank=a.rank, seed=seed)
    blocks = [make(0)]
    warm = 2
    nbytes = blocks[0].bytes(warm + a.steps // 2)       # of the middle one of the timed steps
    plan = plan_rotation(nbytes)
    blocks += [make(seed) for seed in range(1, plan["n_copies"])]
    x = torch.randn(a.batch, blocks[0].qkv.K, device="cuda").to(torch.bfloat16)
    graph = capture(lambda: [block.step(x) for block in blocks], warm=warm)
    us = stats(replay_ms(graph, a.steps))["median"] * 1e3 / len(blocks)
    print(json.dumps({"model": a.model, "fmt": a.fmt, "cache": a.cache, "batch": a.batch, "context": a.context,
                      "adapters": a.adapters, "copies": len(blocks), "llc_safe": plan["llc_safe"], "us_per_step": round(us, 2),
                      "gbps": round(nbytes / us / 1e3, 1)}))
    return 0


if __name__ == "__main__":
    sys.exit(main())
