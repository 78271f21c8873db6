"""Tensor-level API: torch.ops.paia_gemv.* custom ops (torch.library) backed by libpaia_gemv.so.

    from paia_gemv import ops
    y = ops.gemv_fp8(Wq, scale, x)                 # x bf16 [K] or [M,K] (M <= 16) -> y bf16 [N] or [M,N]
    ops.gemv_int4_zp(Wq, s, z, x, bias=b, out=y)   # writes y, allocates nothing

One activation row runs the M = 1 GEMV kernels (`variant` indexes GemvLib.variants / variants_fp8 / variants_int4);
M = 2..16 rows run the small-batch kernels (`variant` indexes GemvLib.variants_batch[fmt]: row-streaming and matrix-core);
-1 is the library's choice, mostly the tile kernel, which has no index.

The ops are registered by libpaia_gemv_torch.so (csrc/torch_ops.cpp); they run on torch's current stream and are
HIP-graph capturable. There is no fallback: if the extension is missing, `load()` raises.
"""
from __future__ import annotations

import os
from pathlib import Path

import torch

_PKG_ROOT = Path(__file__).resolve().parent.parent
_loaded = None


def find_torch_ext() -> str:
    env = os.environ.get("PAIA_GEMV_TORCH_LIB")
    cands = ([env] if env else []) + [str(_PKG_ROOT / "build" / "libpaia_gemv_torch.so")]
    for c in cands:
        if c and os.path.exists(c):
            return c
    raise FileNotFoundError("libpaia_gemv_torch.so not found (run `python paia-project_amd/build.py`). Tried: "
                            + ", ".join(c for c in cands if c))


def load() -> str:
    """Load the torch extension once (it links libpaia_gemv.so from the same directory). Returns its path."""
    global _loaded
    if _loaded is None:
        path = find_torch_ext()
        torch.ops.load_library(path)
        _loaded = path
    return _loaded


def gemv_bf16(W, x, bias=None, variant=-1, out=None):
    load()
    if out is None:
        return torch.ops.paia_gemv.gemv_bf16(W, x, bias, variant)
    torch.ops.paia_gemv.gemv_bf16_out(W, x, bias, variant, out)
    return out


def gemv_fp8(Wq, scale, x, bias=None, variant=-1, out=None):
    load()
    if out is None:
        return torch.ops.paia_gemv.gemv_fp8(Wq, scale, x, bias, variant)
    torch.ops.paia_gemv.gemv_fp8_out(Wq, scale, x, bias, variant, out)
    return out


def gemv_int4(Wq, scales, x, variant=-1, out=None):
    """Reference INT4 format: Wq uint8 [N,K/2] (or int32 [N,K/8]), fp16 scales [N,K/128], zero point 8."""
    load()
    if out is None:
        return torch.ops.paia_gemv.gemv_int4(Wq, scales, x, variant)
    torch.ops.paia_gemv.gemv_int4_out(Wq, scales, x, variant, out)
    return out


def gemv_int4_zp(Wq, scales, zeros, x, bias=None, variant=-1, out=None):
    """Asymmetric INT4: bf16 scales [N,G], zeros uint8 [N,ceil(G/2)], optional bf16 bias [N]."""
    load()
    if out is None:
        return torch.ops.paia_gemv.gemv_int4_zp(Wq, scales, zeros, x, bias, variant)
    torch.ops.paia_gemv.gemv_int4_zp_out(Wq, scales, zeros, x, bias, variant, out)
    return out


def dequant_fp8(Wq, scale):
    load()
    return torch.ops.paia_gemv.dequant_fp8(Wq, scale)


def dequant_int4(Wq, scales):
    load()
    return torch.ops.paia_gemv.dequant_int4(Wq, scales)


def dequant_int4_zp(Wq, scales, zeros):
    load()
    return torch.ops.paia_gemv.dequant_int4_zp(Wq, scales, zeros)


def quantize_fp8_rowwise(W):
    """fp32 W [N,K] on the device -> (q uint8 e4m3 [N,K], scale fp32 [N]) by the HIP quantizer."""
    load()
    return torch.ops.paia_gemv.quantize_fp8_rowwise(W)


def quantize_int4_g128(W):
    """fp32 W [N,K] on the device -> (packed uint8 [N,K/2], scales fp16 [N,K/128]) by the HIP quantizer."""
    load()
    return torch.ops.paia_gemv.quantize_int4_g128(W)


def quantize_int4_zp_g128(W):
    """fp32 W [N,K] on the device -> asymmetric INT4 (packed [N,K/2], scales bf16 [N,G], zeros [N,ceil(G/2)])."""
    load()
    return torch.ops.paia_gemv.quantize_int4_zp_g128(W)


def rope_append(qkv, positions, cos_sin, k_cache, v_cache, slots, num_heads, q_norm=None, k_norm=None, eps=1e-6,
                interleaved=False, k_scale=None, v_scale=None, out=None):
    """Head norms, position rotation and cache write of M tokens in one pass over the fused projection's output.

    qkv bf16 [M, (heads + 2 kv_heads) * head_dim] (rows may be strided) -> rotated q, bf16 [M, heads, head_dim]; k and v
    go to slot slots[m] (int64; negative or past the end: not written) of the cache, in place. The first cos_sin.shape[1]
    dims of each q and k head turn by row positions[m] (int64) of cos_sin (fp32 [context, rotary]: cosines, then sines;
    `rope_table` makes one). q_norm, k_norm: bf16 [head_dim] weights of an RMS norm ahead of the rotation.
    Caches: [pages, kv_heads, page_size, head_dim], bf16, or e4m3 with fp32 [kv_heads] k_scale and v_scale."""
    load()
    args = (qkv, positions, cos_sin, k_cache, v_cache, slots, num_heads, q_norm, k_norm, eps, interleaved, k_scale, v_scale)
    if out is None:
        return torch.ops.paia_gemv.rope_append(*args)
    torch.ops.paia_gemv.rope_append_out(*args, out)
    return out


def rope_table(context, rotary, base=500000.0, inverse_frequencies=None, device=None):
    """The cos_sin argument of rope_append: fp32 [context, rotary], row p = cos(p f), then sin(p f), in 64 bits before the
    rounding. f_i = base^(-2i/rotary), or `inverse_frequencies` [rotary/2] where a model scales them."""
    f = (base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary) if inverse_frequencies is None
         else torch.as_tensor(inverse_frequencies, dtype=torch.float64).cpu())
    angle = torch.arange(context, dtype=torch.float64)[:, None] * f
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device)


def paged_attention(q, k_cache, v_cache, block_table, lens, scale=None, window=0, k_scale=None, v_scale=None,
                    return_lse=False, out=None, workspace=None):
    """Attention of each sequence's newest tokens over the paged cache: out of q's shape, bf16, and with return_lse also
    log sum exp of the scores, fp32 [B, (T,) heads].

    q bf16 [B, heads, head_dim], or [B, T, heads, head_dim] for the T newest tokens (a draft to verify); strided views are
    taken. lens int32 [B] counts each sequence's positions in the cache, the tokens' own included (append first, then
    attend); block_table int32 [B, width] lists its pages, position p on entry p // page_size. Token t sees positions below
    lens[b] - (T-1-t), with a window only the last `window` of them, and none on a page number outside the cache (-1 for
    pages given back); what sees nothing gives 0 (lse -inf). scale defaults to head_dim ** -0.5. Caches as rope_append
    writes them.

    The work is split by the lengths as the GPU finds them, so a captured call may be replayed as they grow.
    `workspace` (any contiguous tensor of `paged_attention_workspace` bytes) avoids an allocation; not to be shared by calls
    that overlap."""
    load()
    args = (q, k_cache, v_cache, block_table, lens, scale, window, k_scale, v_scale, workspace)
    if return_lse:
        if out is not None:
            raise ValueError("paged_attention: out goes without return_lse")
        return torch.ops.paia_gemv.paged_attention_lse(*args)
    if out is None:
        return torch.ops.paia_gemv.paged_attention(*args)
    torch.ops.paia_gemv.paged_attention_out(*args, out)
    return out


def paged_attention_workspace(k_cache, table_width, B, T, num_heads):
    """Bytes that paged_attention's workspace takes for these sizes."""
    load()
    return torch.ops.paia_gemv.paged_attention_workspace(k_cache, table_width, B, T, num_heads)


def lora_add(y, x, A, B, ids, scaling=None, splits=None, out=None, workspace=None):
    """Low-rank adapters of M rows beside a shared projection: y + scaling[a] * (B[a] (A[a] x)), a = ids[m], bf16 [M, N].

    y [M, N] and x [M, K] are bf16 (rows may be strided); A bf16 [adapters, slices * rank, K], B bf16 [adapters, N, rank],
    ids int32 [M] (-1, or any number outside the adapters: the row keeps y), scaling fp32 [adapters]. A fused projection
    names its slices in `splits` (q, k, v or gate, up: their sum is N); each slice has its own `rank` rows of A. Rank and K
    are multiples of 8, rank at most 256. out may be y. Rows that share an adapter read it once for every 16 of them."""
    load()
    args = (y, x, A, B, ids, scaling, splits, workspace)
    if out is None:
        return torch.ops.paia_gemv.lora_add(*args)
    torch.ops.paia_gemv.lora_add_out(*args, out)
    return out


def add_norm(x, residual, norm, post_norm=None, gate=None, weights=None, scale=1.0, eps=1e-6, plus_one=False, out=None,
             residual_out=None):
    """What joins the halves of a layer, in one pass over its rows: (out, residual_out), both [M, D], with

        y = x, or the sum of a token's experts, weights[m, j] x[m, j] over j (x [M, pairs, D], weights fp32 [M, pairs];
            a pair of weight 0 adds nothing, whatever its row holds)
        y = rms(y) * post_norm                      (a norm behind the block, where given)
        residual_out = residual + scale * gate * y  (gate bf16 [D], or [M, D]; residual bf16 or fp32, or None: 0)
        out = rms(residual_out) * norm              (of the sum as it is before its rounding)

    rms(v) = v / sqrt(mean(v^2) + eps). x bf16, norm weights bf16 [D], with plus_one kept less 1. out is bf16, residual_out
    of the residual's type and possibly the residual itself. Rows may be strided; D is a multiple of 8 up to 32768."""
    load()
    args = (x, residual, norm, post_norm, gate, weights, scale, eps, plus_one)
    if out is None and residual_out is None:
        return torch.ops.paia_gemv.add_norm(*args)
    if out is None:
        out = torch.empty(x.shape[0], x.shape[-1], dtype=torch.bfloat16, device=x.device)
    if residual_out is None:
        residual_out = torch.empty(x.shape[0], x.shape[-1], device=x.device,
                                   dtype=torch.bfloat16 if residual is None else residual.dtype)
    torch.ops.paia_gemv.add_norm_out(*args, out, residual_out)
    return out, residual_out


def route_experts(logits, k, bias=None, scoring="softmax", renormalize=True, scale=1.0, workspace=None):
    """Each token's k experts and the order that the experts' products take them in: (ids int32 [M, k], weights fp32 [M, k],
    order int32 [M * k], offsets int32 [experts + 1]).

    logits bf16 or fp32 [M, experts] (rows may be strided). The experts of the largest logits, or with scoring "sigmoid" of
    the largest sigmoid(logit) + bias (fp32 [experts]); equal ones by the lower index. weights are scale times the softmax
    over the row, or the sigmoid (without the bias), with renormalize divided by their sum over the token's k. An expert whose
    logit or bias is -inf or NaN is closed; where fewer than k are open the ids end with -1, of weight 0 (a row of -inf is a
    token that is not there). order lists the pairs m * k + j by expert, offsets[e] is where expert e's begin, and what comes
    from offsets[-1] on has no expert. experts up to 1024, k up to 64."""
    load()
    return torch.ops.paia_gemv.route_experts(logits, k, bias, scoring, renormalize, scale, workspace)


def expert_order(ids, experts, workspace=None):
    """route_experts' (order, offsets) for ids int32 [M, k] chosen otherwise (outside [0, experts): no expert)."""
    load()
    return torch.ops.paia_gemv.expert_order(ids, experts, workspace)


def route_experts_workspace(M, experts, k):
    """Bytes that the workspace of route_experts and expert_order takes for these sizes (0 for few tokens)."""
    load()
    return torch.ops.paia_gemv.route_experts_workspace(M, experts, k)


def experts_bf16(W, x, order, offsets, bias=None, gated=False, out=None):
    """Products with the experts' matrices, W bf16 [experts, N, K]: out[p] = W[e] x[p // (pairs // rows)] (+ bias[e]) for every
    pair p of token and expert, bf16 [pairs, N].

    order and offsets as route_experts makes them. x bf16 [rows, K] (rows may be strided) has a row for each token, whose
    pairs share it, or for each pair (the down projection). gated: an expert's rows are N/2 gates and N/2 values,
    out = silu(gate) * value, [pairs, N/2]. bias bf16 [experts, N]. Pairs without an expert give 0. Any number of tokens:
    a few are bound by reading the chosen experts once, many run on the matrix cores."""
    load()
    if out is None:
        return torch.ops.paia_gemv.experts_bf16(W, x, order, offsets, bias, gated)
    torch.ops.paia_gemv.experts_bf16_out(W, x, order, offsets, bias, gated, out)
    return out


def experts_fp8(Wq, scale, x, order, offsets, bias=None, gated=False, out=None):
    """experts_bf16 with e4m3 weights [experts, N, K] and fp32 scales [experts, N]."""
    load()
    if out is None:
        return torch.ops.paia_gemv.experts_fp8(Wq, scale, x, order, offsets, bias, gated)
    torch.ops.paia_gemv.experts_fp8_out(Wq, scale, x, order, offsets, bias, gated, out)
    return out


def experts_int4(Wq, scales, x, order, offsets, gated=False, out=None):
    """experts_bf16 with the reference's INT4 format: Wq uint8 [experts, N, K/2] (or int32 [.., K/8]), fp16 scales
    [experts, N, K/128], zero point 8."""
    load()
    if out is None:
        return torch.ops.paia_gemv.experts_int4(Wq, scales, x, order, offsets, gated)
    torch.ops.paia_gemv.experts_int4_out(Wq, scales, x, order, offsets, gated, out)
    return out


def experts_int4_zp(Wq, scales, zeros, x, order, offsets, bias=None, gated=False, out=None):
    """experts_bf16 with asymmetric INT4: bf16 scales [experts, N, G], zeros uint8 [experts, N, ceil(G/2)]."""
    load()
    if out is None:
        return torch.ops.paia_gemv.experts_int4_zp(Wq, scales, zeros, x, order, offsets, bias, gated)
    torch.ops.paia_gemv.experts_int4_zp_out(Wq, scales, zeros, x, order, offsets, bias, gated, out)
    return out
