"""ctypes loader for libpaia_gemv.so, the gfx950 HIP build (no torch ABI dependency in the library itself).

Drop-in for src/paia_gemv/loader.py:12-109: same `find_lib`, `current_raw_stream`, `GemvLib` (attributes `path`,
`n_variants`, `variants`, `variants_fp8`, `variants_int4`; methods `bf16`, `fp8`, `int4`, `int4_naive`,
`int4_unfused`) and `load_lib`. Pointers are plain ints; a nonzero return code raises RuntimeError. Launches go on
torch's current stream, so calls can be captured into a HIP graph (torch.cuda.CUDAGraph on ROCm).

Additions for the gfx950 build: `bf16_bias`, `fp8_bias`, `int4_zp` (asymmetric INT4 with optional bias),
`dequant_fp8`, `dequant_int4`, `dequant_int4_zp`, `quantize_fp8_rowwise`, `quantize_int4_g128`,
`quantize_int4_zp_g128`, `pick_variant`, `launch_kind`, `build_info`, and between the projections of a decode step
`rope_append` and `paged_attention` (on a `KVCache` description of the paged cache), beside them `lora_add`; for a layer's
feed-forward half with experts `add_norm`, `route_experts`, `expert_order` and `experts_bf16/fp8/int4/int4_zp`.
"""
from __future__ import annotations

import ctypes
import os
import platform
from pathlib import Path

_PKG_ROOT = Path(__file__).resolve().parent.parent       # paia-project_amd/


def find_lib() -> str:
    """PAIA_GEMV_LIB, else <pkg>/build/<machine>/libpaia_gemv.so, else <pkg>/build/libpaia_gemv.so."""
    env = os.environ.get("PAIA_GEMV_LIB")
    cands = [env] if env else []
    cands += [str(_PKG_ROOT / "build" / platform.machine() / "libpaia_gemv.so"),
              str(_PKG_ROOT / "build" / "libpaia_gemv.so")]
    for c in cands:
        if c and os.path.exists(c):
            return c
    raise FileNotFoundError("libpaia_gemv.so not found (run `python paia-project_amd/build.py`, or set "
                            "PAIA_GEMV_LIB). Tried: " + ", ".join(c for c in cands if c))


def current_raw_stream():
    import torch
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
_F = ctypes.c_float
KINDS = {"bf16": 0, "fp8": 1, "int4": 2, "int4zp": 3}


class KVCache(ctypes.Structure):
    """paia_kv_cache: device addresses (k_scale, v_scale fp32 [kv_heads] or None) and the strides, in elements, of page,
    head and position. Positions of one head are together by default: [pages, kv_heads, page_size, head_dim]."""
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("k_strides", _L * 3), ("v_strides", _L * 3),
                ("pages", _I), ("page_size", _I), ("kv_heads", _I), ("head_dim", _I), ("fp8", _I)]

    def __init__(self, k_ptr, v_ptr, pages, page_size, kv_heads, head_dim, fp8=False, k_scale_ptr=None, v_scale_ptr=None,
                 k_strides=None, v_strides=None):
        plain = (kv_heads * page_size * head_dim, page_size * head_dim, head_dim)
        super().__init__(k_ptr, v_ptr, k_scale_ptr, v_scale_ptr, (_L * 3)(*(k_strides or plain)),
                         (_L * 3)(*(v_strides or plain)), pages, page_size, kv_heads, head_dim, int(fp8))


class GemvLib:
    CODES = "-1: no such variant; -2: shape or alignment outside the contract; > 0: HIP error"

    def __init__(self, path=None):
        self.path = path or find_lib()
        lib = ctypes.CDLL(self.path)
        sig = {
            "paia_gemv_bf16": [_P, _P, _P, _I, _I, _I, _P],
            "paia_gemv_bf16_bias": [_P, _P, _P, _P, _I, _I, _I, _P],
            "paia_gemv_fp8": [_P, _P, _P, _P, _I, _I, _I, _P],
            "paia_gemv_fp8_bias": [_P, _P, _P, _P, _P, _I, _I, _I, _P],
            "paia_gemv_int4": [_P, _P, _P, _P, _I, _I, _I, _P],
            "paia_gemv_int4_naive": [_P, _P, _P, _P, _I, _I, _P],
            "paia_gemv_int4_unfused": [_P, _P, _P, _P, _P, _I, _I, _P],
            "paia_gemv_int4_unfused_noalloc": [_P, _P, _P, _P, _I, _I, _P],
            "paia_gemv_int4_zp": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P],
            "paia_dequant_fp8": [_P, _P, _P, _I, _I, _P],
            "paia_dequant_int4": [_P, _P, _P, _I, _I, _P],
            "paia_dequant_int4_zp": [_P, _P, _P, _P, _I, _I, _P],
            "paia_quantize_fp8_rowwise": [_P, _P, _P, _I, _I, _P],
            "paia_quantize_int4_g128": [_P, _P, _P, _I, _I, _P],
            "paia_quantize_int4_zp_g128": [_P, _P, _P, _P, _I, _I, _P],
            "paia_gemv_pick_variant": [_I, _I, _I],
            "paia_gemv_launch_kind": [_I, _I, _I, _I],
            "paia_gemv_bf16_variant_count": [],
            "paia_gemv_bf16_variant_info": [_I] + [ctypes.POINTER(_I)] * 5,
            "paia_gemv_batch_variant_count": [_I],
            "paia_gemv_batch_variant_info": [_I, _I] + [ctypes.POINTER(_I)] * 5,
            "paia_gemv_batch_pick_variant": [_I, _I, _I, _I],
            "paia_gemv_batch_bf16": [_P, _P, _P, _P, _I, _I, _I, _I, _P],
            "paia_gemv_batch_fp8": [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
            "paia_gemv_batch_int4": [_P, _P, _P, _P, _I, _I, _I, _I, _P],
            "paia_gemv_batch_int4_zp": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
            "paia_rope_append": [_P, _L, _P, _P, _I, _I, _I, _P, _P, _F, _P, ctypes.POINTER(KVCache), _P, _I, _I, _P],
            "paia_paged_attention": [_P, ctypes.POINTER(_L), ctypes.POINTER(KVCache), _P, _L, _I, _P, _F, _I, _P, _P, _I,
                                     _I, _I, _P, _L, _P],
            "paia_lora_add": [_P, _L, _P, _L, _P, _P, _P, _P, _P, _L, _I, _I, _I, ctypes.POINTER(_I), _I, _I, _P, _L, _P],
            "paia_add_norm": [_P, _L, _P, _L, _I, _P, _L, _I, _P, _P, _L, _F, _P, _I, _F, _P, _L, _P, _L, _I, _I, _P],
            "paia_route_experts": [_P, _I, _L, _P, _I, _I, _F, _P, _P, _P, _P, _I, _I, _I, _P, _L, _P],
            "paia_expert_order": [_P, _P, _P, _I, _I, _I, _P, _L, _P],
            "paia_experts_bf16": [_P, _P, _L, _I, _P, _P, _P, _P, _L, _I, _I, _I, _I, _I, _P],
            "paia_experts_fp8": [_P, _P, _P, _L, _I, _P, _P, _P, _P, _L, _I, _I, _I, _I, _I, _P],
            "paia_experts_int4": [_P, _P, _P, _L, _I, _P, _P, _P, _L, _I, _I, _I, _I, _I, _P],
            "paia_experts_int4_zp": [_P, _P, _P, _P, _L, _I, _P, _P, _P, _P, _L, _I, _I, _I, _I, _I, _P],
        }
        for name, argtypes in sig.items():
            fn = getattr(lib, name)
            fn.restype = _I
            fn.argtypes = argtypes
        lib.paia_paged_attention_workspace.restype = _L
        lib.paia_paged_attention_workspace.argtypes = [ctypes.POINTER(KVCache), _I, _I, _I, _I]
        lib.paia_lora_add_workspace.restype = _L
        lib.paia_lora_add_workspace.argtypes = [_I, _I, _I, ctypes.POINTER(_I), _I]
        lib.paia_route_experts_workspace.restype = _L
        lib.paia_route_experts_workspace.argtypes = [_I, _I, _I]
        lib.paia_gemv_build_info.restype = ctypes.c_char_p
        lib.paia_gemv_build_info.argtypes = []
        self.variants_fp8 = self._qvariants(lib, "fp8")
        self.variants_int4 = self._qvariants(lib, "int4")
        self._lib = lib
        self._fn = lib.paia_gemv_bf16
        self.n_variants = lib.paia_gemv_bf16_variant_count()
        self.variants = []
        for v in range(self.n_variants):
            R, U, W, S, H = (_I() for _ in range(5))
            assert lib.paia_gemv_bf16_variant_info(v, *map(ctypes.byref, (R, U, W, S, H))) == 0
            self.variants.append({"id": v, "R": R.value, "U": U.value, "W": W.value, "S": S.value, "H": H.value})
        self.variants_batch = {}
        for kind, k in KINDS.items():
            vs = []
            for v in range(lib.paia_gemv_batch_variant_count(k)):
                P, U, W, S, X = (_I() for _ in range(5))
                assert lib.paia_gemv_batch_variant_info(k, v, *map(ctypes.byref, (P, U, W, S, X))) == 0
                vs.append({"id": v, "P": P.value, "U": U.value, "W": W.value, "S": S.value, "X": X.value})
            self.variants_batch[kind] = vs

    @staticmethod
    def _qvariants(lib, kind):
        count = getattr(lib, f"paia_gemv_{kind}_variant_count")
        count.restype = _I
        count.argtypes = []
        info = getattr(lib, f"paia_gemv_{kind}_variant_info")
        info.restype = _I
        info.argtypes = [_I] + [ctypes.POINTER(_I)] * 4
        out = []
        for v in range(count()):
            R, U, W, H = (_I() for _ in range(4))
            assert info(v, *map(ctypes.byref, (R, U, W, H))) == 0
            out.append({"id": v, "R": R.value, "U": U.value, "W": W.value, "S": 0, "H": H.value})
        return out

    @classmethod
    def _check(cls, rc, what):
        if rc != 0:
            raise RuntimeError(f"{what} returned {rc} ({cls.CODES})")

    @staticmethod
    def _st(stream):
        return current_raw_stream() if stream is None else stream

    # ---- reference surface -------------------------------------------------------------------------------
    def bf16(self, W_ptr, x_ptr, y_ptr, N, K, variant, stream=None):
        """BF16 weights: the output vector (N bf16 values) from the row-major N x K matrix and the K-vector, each
        passed as a device address (int)."""
        rc = self._fn(W_ptr, x_ptr, y_ptr, N, K, variant, self._st(stream))
        if rc != 0:
            raise RuntimeError(f"paia_gemv_bf16 returned {rc} for N={N} K={K} variant {variant} "
                               "(-1: no such variant; -2: K not a multiple of 8 or a pointer not 16-byte aligned; "
                               "> 0: HIP error)")

    def fp8(self, Wq_ptr, scale_ptr, x_ptr, y_ptr, N, K, variant, stream=None):
        """FP8 weights: one e4m3fn byte per weight (N x K), one fp32 scale per output row; bf16 x and y; K a
        multiple of 16."""
        self._check(self._lib.paia_gemv_fp8(Wq_ptr, scale_ptr, x_ptr, y_ptr, N, K, variant, self._st(stream)),
                    "paia_gemv_fp8")

    def int4(self, Wq_ptr, scales_ptr, x_ptr, y_ptr, N, K, variant, stream=None):
        """INT4 weights, two per byte (N x K/2), zero point 8, one fp16 scale per 128 columns of a row; K a multiple
        of 128. The fused kernel."""
        self._check(self._lib.paia_gemv_int4(Wq_ptr, scales_ptr, x_ptr, y_ptr, N, K, variant, self._st(stream)),
                    "paia_gemv_int4")

    def int4_naive(self, Wq_ptr, scales_ptr, x_ptr, y_ptr, N, K, stream=None):
        self._check(self._lib.paia_gemv_int4_naive(Wq_ptr, scales_ptr, x_ptr, y_ptr, N, K, self._st(stream)),
                    "paia_gemv_int4_naive")

    def int4_unfused(self, Wq_ptr, scales_ptr, x_ptr, y_ptr, scratch_ptr, N, K, stream=None):
        self._check(self._lib.paia_gemv_int4_unfused(Wq_ptr, scales_ptr, x_ptr, y_ptr, scratch_ptr, N, K,
                                                     self._st(stream)), "paia_gemv_int4_unfused")

    # ---- gfx950 additions --------------------------------------------------------------------------------
    def int4_unfused_noalloc(self, Wq_ptr, scales_ptr, x_ptr, y_ptr, N, K, stream=None):
        """The unfused control without a workspace argument: the library's static device scratch (for callers that
        cannot allocate; calls that overlap on one GPU race)."""
        self._check(self._lib.paia_gemv_int4_unfused_noalloc(Wq_ptr, scales_ptr, x_ptr, y_ptr, N, K, self._st(stream)),
                    "paia_gemv_int4_unfused_noalloc")

    def bf16_bias(self, W_ptr, x_ptr, bias_ptr, y_ptr, N, K, variant, stream=None):
        self._check(self._lib.paia_gemv_bf16_bias(W_ptr, x_ptr, bias_ptr, y_ptr, N, K, variant, self._st(stream)),
                    "paia_gemv_bf16_bias")

    def fp8_bias(self, Wq_ptr, scale_ptr, x_ptr, bias_ptr, y_ptr, N, K, variant, stream=None):
        self._check(self._lib.paia_gemv_fp8_bias(Wq_ptr, scale_ptr, x_ptr, bias_ptr, y_ptr, N, K, variant,
                                                 self._st(stream)), "paia_gemv_fp8_bias")

    def int4_zp(self, Wq_ptr, scales_ptr, zeros_ptr, x_ptr, bias_ptr, y_ptr, N, K, variant, stream=None):
        """Asymmetric INT4: scales bf16 [N,G], zeros [N,ceil(G/2)] (2 nibbles/byte), bias bf16 [N] or None."""
        self._check(self._lib.paia_gemv_int4_zp(Wq_ptr, scales_ptr, zeros_ptr, x_ptr, bias_ptr, y_ptr, N, K, variant,
                                                self._st(stream)), "paia_gemv_int4_zp")

    def dequant_fp8(self, Wq_ptr, scale_ptr, out_ptr, N, K, stream=None):
        self._check(self._lib.paia_dequant_fp8(Wq_ptr, scale_ptr, out_ptr, N, K, self._st(stream)), "paia_dequant_fp8")

    def dequant_int4(self, Wq_ptr, scales_ptr, out_ptr, N, K, stream=None):
        self._check(self._lib.paia_dequant_int4(Wq_ptr, scales_ptr, out_ptr, N, K, self._st(stream)),
                    "paia_dequant_int4")

    def dequant_int4_zp(self, Wq_ptr, scales_ptr, zeros_ptr, out_ptr, N, K, stream=None):
        self._check(self._lib.paia_dequant_int4_zp(Wq_ptr, scales_ptr, zeros_ptr, out_ptr, N, K, self._st(stream)),
                    "paia_dequant_int4_zp")

    def quantize_fp8_rowwise(self, W_ptr, q_ptr, scale_ptr, N, K, stream=None):
        """fp32 W [N,K] -> e4m3 q [N,K], fp32 scale [N] on the device (quant.py:8-13 semantics)."""
        self._check(self._lib.paia_quantize_fp8_rowwise(W_ptr, q_ptr, scale_ptr, N, K, self._st(stream)),
                    "paia_quantize_fp8_rowwise")

    def quantize_int4_g128(self, W_ptr, packed_ptr, scales_ptr, N, K, stream=None):
        """fp32 W [N,K] -> packed [N,K/2], fp16 scales [N,K/128] on the device (quant.py:20-31 semantics)."""
        self._check(self._lib.paia_quantize_int4_g128(W_ptr, packed_ptr, scales_ptr, N, K, self._st(stream)),
                    "paia_quantize_int4_g128")

    def quantize_int4_zp_g128(self, W_ptr, packed_ptr, scales_ptr, zeros_ptr, N, K, stream=None):
        """fp32 W [N,K] -> asymmetric INT4: packed [N,K/2], bf16 scales [N,G], zeros [N,ceil(G/2)] on the device."""
        self._check(self._lib.paia_quantize_int4_zp_g128(W_ptr, packed_ptr, scales_ptr, zeros_ptr, N, K,
                                                         self._st(stream)), "paia_quantize_int4_zp_g128")

    def pick_variant(self, kind, N, K):
        """Library's per-shape variant: kind 'bf16' | 'fp8' | 'int4' | 'int4zp' (an index of variants_int4)."""
        return self._lib.paia_gemv_pick_variant(KINDS[kind], N, K)

    # ---- small batch (M = 1..16 activation rows, x [M,K] and y [M,N] bf16 row-major) -------------------------
    KERNELS = ("gemv_kernel", "gemv_kernel43", "gemv_kernel_xg", "gemv_kernel_dr", "gemv_kernel43_dr")

    def launch_kind(self, kind, N, K, variant):
        """The kernel a call of `variant` runs at (N, K), as a profiler names it: "gemv_kernel", "gemv_kernel43" (INT4
        launches with few weight loads per wave) or "gemv_kernel_xg" (K beyond the LDS staging)."""
        k = self._lib.paia_gemv_launch_kind(KINDS[kind], N, K, variant)
        if k < 0:
            raise ValueError(f"paia_gemv_launch_kind({kind}, {N}, {K}, {variant}) returned {k}")
        return self.KERNELS[k]

    def batch_pick_variant(self, kind, M, N, K):
        """The best entry of variants_batch[kind] for the shape; -1 if M is out of range. A call whose variant is left to
        the library may instead run the tile kernel, which has no entry."""
        return self._lib.paia_gemv_batch_pick_variant(KINDS[kind], M, N, K)

    def batch_bf16(self, W_ptr, x_ptr, bias_ptr, y_ptr, M, N, K, variant=-1, stream=None):
        self._check(self._lib.paia_gemv_batch_bf16(W_ptr, x_ptr, bias_ptr, y_ptr, M, N, K, variant, self._st(stream)),
                    "paia_gemv_batch_bf16")

    def batch_fp8(self, Wq_ptr, scale_ptr, x_ptr, bias_ptr, y_ptr, M, N, K, variant=-1, stream=None):
        self._check(self._lib.paia_gemv_batch_fp8(Wq_ptr, scale_ptr, x_ptr, bias_ptr, y_ptr, M, N, K, variant,
                                                  self._st(stream)), "paia_gemv_batch_fp8")

    def batch_int4(self, Wq_ptr, scales_ptr, x_ptr, y_ptr, M, N, K, variant=-1, stream=None):
        self._check(self._lib.paia_gemv_batch_int4(Wq_ptr, scales_ptr, x_ptr, y_ptr, M, N, K, variant,
                                                   self._st(stream)), "paia_gemv_batch_int4")

    def batch_int4_zp(self, Wq_ptr, scales_ptr, zeros_ptr, x_ptr, bias_ptr, y_ptr, M, N, K, variant=-1, stream=None):
        self._check(self._lib.paia_gemv_batch_int4_zp(Wq_ptr, scales_ptr, zeros_ptr, x_ptr, bias_ptr, y_ptr, M, N, K,
                                                      variant, self._st(stream)), "paia_gemv_batch_int4_zp")

    # ---- between the projections of a decode step -------------------------------------------------------------
    def rope_append(self, qkv_ptr, qkv_stride, positions_ptr, cos_sin_ptr, context, rotary, slots_ptr, cache, q_ptr, M,
                    heads, q_norm_ptr=None, k_norm_ptr=None, eps=1e-6, interleaved=False, stream=None):
        """Head norms, rotation and cache write of M tokens' q|k|v rows (bf16, qkv_stride elements apart): rotated q
        [M, heads, head_dim] to q_ptr, k and v to their slots (int64) of `cache` (a KVCache)."""
        self._check(self._lib.paia_rope_append(qkv_ptr, qkv_stride, positions_ptr, cos_sin_ptr, context, rotary,
                                               int(interleaved), q_norm_ptr, k_norm_ptr, eps, slots_ptr,
                                               ctypes.byref(cache), q_ptr, M, heads, self._st(stream)),
                    "paia_rope_append")

    def paged_attention_workspace(self, cache, table_width, B, T, heads):
        """Bytes of device memory that paged_attention takes as its workspace."""
        need = self._lib.paia_paged_attention_workspace(ctypes.byref(cache), table_width, B, T, heads)
        self._check(min(need, 0), "paia_paged_attention_workspace")
        return need

    def paged_attention(self, q_ptr, cache, table_ptr, table_width, lens_ptr, out_ptr, B, T, heads, scale, window=0,
                        lse_ptr=None, workspace_ptr=None, workspace_bytes=0, q_strides=None, table_stride=None,
                        stream=None):
        """Attention of each sequence's T newest tokens (q bf16 [B, T, heads, head_dim], or strides in elements) over
        `cache` (a KVCache) through the int32 block table and lens."""
        D = cache.head_dim
        strides = (_L * 3)(*(q_strides or (T * heads * D, heads * D, D)))
        self._check(self._lib.paia_paged_attention(q_ptr, strides, ctypes.byref(cache), table_ptr,
                                                   table_width if table_stride is None else table_stride, table_width,
                                                   lens_ptr, scale, window, out_ptr, lse_ptr, B, T, heads, workspace_ptr,
                                                   workspace_bytes, self._st(stream)), "paia_paged_attention")

    def lora_add_workspace(self, M, K, rank, splits):
        """Bytes of device memory that lora_add takes as its workspace (0 for few rows of a low rank)."""
        need = self._lib.paia_lora_add_workspace(M, K, rank, (_I * len(splits))(*splits), len(splits))
        self._check(min(need, 0), "paia_lora_add_workspace")
        return need

    def lora_add(self, y_ptr, x_ptr, A_ptr, B_ptr, ids_ptr, scaling_ptr, out_ptr, M, K, rank, splits, adapters,
                 workspace_ptr, workspace_bytes, y_stride=None, x_stride=None, out_stride=None, stream=None):
        """out [M, sum(splits)] = y + the rows' adapters; see ops.lora_add. Strides in elements, rows contiguous by
        default."""
        N = sum(splits)
        self._check(self._lib.paia_lora_add(y_ptr, N if y_stride is None else y_stride, x_ptr,
                                            K if x_stride is None else x_stride, A_ptr, B_ptr, ids_ptr, scaling_ptr,
                                            out_ptr, N if out_stride is None else out_stride, M, K, rank,
                                            (_I * len(splits))(*splits), len(splits), adapters, workspace_ptr,
                                            workspace_bytes, self._st(stream)), "paia_lora_add")

    def add_norm(self, x_ptr, residual_ptr, norm_ptr, out_ptr, residual_out_ptr, M, D, weights_ptr=None, pairs=0,
                 post_norm_ptr=None, gate_ptr=None, gate_stride=0, scale=1.0, eps=1e-6, plus_one=False, residual_fp32=False,
                 x_stride=None, pair_stride=None, residual_stride=None, out_stride=None, residual_out_stride=None,
                 stream=None):
        """out, residual_out [M, D] of x [M, D] or [M, pairs, D]; see ops.add_norm. Strides in elements, all contiguous by
        default; gate_stride 0: one row of gates for all."""
        d = lambda stride, plain: plain if stride is None else stride  # noqa: E731
        self._check(self._lib.paia_add_norm(x_ptr, d(x_stride, max(1, pairs) * D), weights_ptr, d(pair_stride, D), pairs,
                                            residual_ptr, d(residual_stride, D), int(residual_fp32), post_norm_ptr, gate_ptr,
                                            gate_stride, scale, norm_ptr, int(plus_one), eps, out_ptr, d(out_stride, D),
                                            residual_out_ptr, d(residual_out_stride, D), M, D, self._st(stream)),
                    "paia_add_norm")

    def route_experts_workspace(self, M, experts, k):
        """Bytes of device memory that route_experts and expert_order take as their workspace (0 for few tokens)."""
        need = self._lib.paia_route_experts_workspace(M, experts, k)
        self._check(min(need, 0), "paia_route_experts_workspace")
        return need

    def route_experts(self, logits_ptr, ids_ptr, weights_ptr, order_ptr, offsets_ptr, M, experts, k, workspace_ptr=None,
                      workspace_bytes=0, bias_ptr=None, sigmoid=False, renormalize=True, scale=1.0, fp32=False,
                      logits_stride=None, stream=None):
        """Each token's experts and their order; see ops.route_experts."""
        self._check(self._lib.paia_route_experts(logits_ptr, int(fp32), experts if logits_stride is None else logits_stride,
                                                 bias_ptr, int(sigmoid), int(renormalize), scale, ids_ptr, weights_ptr,
                                                 order_ptr, offsets_ptr, M, experts, k, workspace_ptr, workspace_bytes,
                                                 self._st(stream)), "paia_route_experts")

    def expert_order(self, ids_ptr, order_ptr, offsets_ptr, M, experts, k, workspace_ptr=None, workspace_bytes=0,
                     stream=None):
        self._check(self._lib.paia_expert_order(ids_ptr, order_ptr, offsets_ptr, M, experts, k, workspace_ptr,
                                                workspace_bytes, self._st(stream)), "paia_expert_order")

    def _experts(self, name, weights, x_ptr, x_rows, order_ptr, offsets_ptr, bias, out_ptr, experts, N, K, pairs, gated,
                 x_stride, out_stride, stream):
        cols = N // 2 if gated else N
        self._check(getattr(self._lib, name)(*weights, x_ptr, K if x_stride is None else x_stride, x_rows, order_ptr,
                                             offsets_ptr, *bias, out_ptr, cols if out_stride is None else out_stride, experts,
                                             N, K, pairs, int(gated), self._st(stream)), name)

    def experts_bf16(self, W_ptr, x_ptr, x_rows, order_ptr, offsets_ptr, out_ptr, experts, N, K, pairs, bias_ptr=None,
                     gated=False, x_stride=None, out_stride=None, stream=None):
        """out [pairs, N] (gated: N // 2) of the experts' matrices and the rows of x; see ops.experts_bf16."""
        self._experts("paia_experts_bf16", (W_ptr,), x_ptr, x_rows, order_ptr, offsets_ptr, (bias_ptr,), out_ptr, experts, N,
                      K, pairs, gated, x_stride, out_stride, stream)

    def experts_fp8(self, Wq_ptr, scale_ptr, x_ptr, x_rows, order_ptr, offsets_ptr, out_ptr, experts, N, K, pairs,
                    bias_ptr=None, gated=False, x_stride=None, out_stride=None, stream=None):
        self._experts("paia_experts_fp8", (Wq_ptr, scale_ptr), x_ptr, x_rows, order_ptr, offsets_ptr, (bias_ptr,), out_ptr,
                      experts, N, K, pairs, gated, x_stride, out_stride, stream)

    def experts_int4(self, Wq_ptr, scales_ptr, x_ptr, x_rows, order_ptr, offsets_ptr, out_ptr, experts, N, K, pairs,
                     gated=False, x_stride=None, out_stride=None, stream=None):
        self._experts("paia_experts_int4", (Wq_ptr, scales_ptr), x_ptr, x_rows, order_ptr, offsets_ptr, (), out_ptr, experts,
                      N, K, pairs, gated, x_stride, out_stride, stream)

    def experts_int4_zp(self, Wq_ptr, scales_ptr, zeros_ptr, x_ptr, x_rows, order_ptr, offsets_ptr, out_ptr, experts, N, K,
                        pairs, bias_ptr=None, gated=False, x_stride=None, out_stride=None, stream=None):
        self._experts("paia_experts_int4_zp", (Wq_ptr, scales_ptr, zeros_ptr), x_ptr, x_rows, order_ptr, offsets_ptr,
                      (bias_ptr,), out_ptr, experts, N, K, pairs, gated, x_stride, out_stride, stream)

    def build_info(self):
        return self._lib.paia_gemv_build_info().decode()


_lib = None


def load_lib():
    global _lib
    if _lib is None:
        _lib = GemvLib()
    return _lib
