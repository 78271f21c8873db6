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
