"""Host-side checks of the entry points of a layer's feed-forward half: every call below returns from them, nothing is launched (no
GPU needed)."""
import ctypes

import pytest
import torch

A = 1 << 20      # a 16-byte-aligned address, never dereferenced


def norm(lib, **change):
    a = dict(x=A, xs=64, w=None, ps=0, pairs=0, res=A, rs=64, wide=0, post=None, gate=None, gs=0, scale=1.0, norm=A, one=0,
             eps=1e-6, out=A, os=64, rout=A, ros=64, M=4, D=64)
    a.update(change)
    return lib._lib.paia_add_norm(*[a[k] for k in ("x", "xs", "w", "ps", "pairs", "res", "rs", "wide", "post", "gate", "gs", "scale",
                                                   "norm", "one", "eps", "out", "os", "rout", "ros", "M", "D")], None)


def test_add_norm_refusals(gemv_lib):
    for bad in (dict(x=None), dict(x=A + 8), dict(xs=60), dict(xs=-64), dict(w=A), dict(pairs=2), dict(pairs=2, w=A + 2),
                dict(pairs=-1), dict(pairs=2, w=A, ps=4), dict(res=A + 2), dict(rs=4), dict(wide=2), dict(post=A + 8),
                dict(gate=A + 4), dict(gs=12), dict(norm=None), dict(norm=A + 8), dict(one=2), dict(eps=-1.0),
                dict(eps=float("nan")), dict(out=None), dict(out=A + 8), dict(os=56), dict(rout=A + 4), dict(ros=56), dict(M=-1),
                dict(D=0), dict(D=60), dict(D=32776)):
        assert norm(gemv_lib, **bad) == -2, bad
    assert norm(gemv_lib, M=0) == 0


def route(lib, **change):
    a = dict(logits=A, wide=0, stride=64, bias=None, sigmoid=0, renorm=1, scale=1.0, ids=A, w=A, order=A, off=A, M=100, E=64, k=4,
             space=A, bytes=1 << 40)
    a.update(change)
    return lib._lib.paia_route_experts(*[a[k] for k in ("logits", "wide", "stride", "bias", "sigmoid", "renorm", "scale", "ids", "w",
                                                        "order", "off", "M", "E", "k", "space", "bytes")], None)


def test_route_experts_refusals(gemv_lib):
    for bad in (dict(logits=None), dict(logits=A + 1), dict(logits=A + 2, wide=1), dict(wide=2), dict(stride=-1), dict(bias=A),
                dict(bias=A + 2, sigmoid=1), dict(sigmoid=2), dict(renorm=2), dict(ids=None), dict(ids=A + 2), dict(w=None),
                dict(w=A + 2), dict(order=None), dict(order=A + 1), dict(off=None), dict(off=A + 2), dict(M=-1), dict(E=0),
                dict(E=1025), dict(k=0), dict(k=65, E=128), dict(k=65), dict(M=1 << 24), dict(space=None), dict(space=A + 4),
                dict(bytes=100)):
        assert route(gemv_lib, **bad) == -2, bad
    need = gemv_lib._lib.paia_route_experts_workspace
    assert need(1, 64, 4) == 0 and need(32, 1024, 64) == 0
    assert 0 < need(33, 64, 4) < need(4096, 64, 4) == need(100000, 64, 4)       # bounded by the blocks, not by the tokens
    for bad in ((-1, 64, 4), (4, 0, 4), (4, 1025, 4), (4, 64, 0), (4, 64, 65), (1 << 24, 64, 4)):
        assert need(*bad) == -2
        with pytest.raises(RuntimeError, match="-2"):
            gemv_lib.route_experts_workspace(*bad)


def order(lib, **change):
    a = dict(ids=A, order=A, off=A, M=100, E=64, k=4, space=A, bytes=1 << 40)
    a.update(change)
    return lib._lib.paia_expert_order(*[a[k] for k in ("ids", "order", "off", "M", "E", "k", "space", "bytes")], None)


def test_expert_order_refusals(gemv_lib):
    for bad in (dict(ids=None), dict(ids=A + 2), dict(order=None), dict(order=A + 2), dict(off=None), dict(off=A + 1), dict(M=-1),
                dict(E=0), dict(E=1025), dict(k=0), dict(k=65), dict(space=None), dict(space=A + 8), dict(bytes=16)):
        assert order(gemv_lib, **bad) == -2, bad


def experts(lib, fmt, **change):
    a = dict(W=A, meta=A, zeros=A, x=A, xs=256, rows=4, order=A, off=A, bias=None, out=A, os=64, E=8, N=64, K=256, pairs=8, gated=0)
    a.update(change)
    weights = {"bf16": ("W",), "fp8": ("W", "meta"), "int4": ("W", "meta"), "int4_zp": ("W", "meta", "zeros")}[fmt]
    bias = () if fmt == "int4" else ("bias",)
    names = (*weights, "x", "xs", "rows", "order", "off", *bias, "out", "os", "E", "N", "K", "pairs", "gated")
    return getattr(lib._lib, f"paia_experts_{fmt}")(*[a[k] for k in names], None)


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int4", "int4_zp"])
def test_experts_refusals(gemv_lib, fmt):
    bad = [dict(W=None), dict(W=A + 8), dict(x=None), dict(x=A + 8), dict(xs=252), dict(xs=248), dict(xs=-256), dict(rows=0),
           dict(rows=3), dict(rows=-1), dict(order=None), dict(order=A + 2), dict(off=None), dict(off=A + 2), dict(out=None),
           dict(out=A + 1), dict(os=63), dict(os=-64), dict(E=0), dict(E=1025), dict(N=0), dict(K=0), dict(K=(1 << 25) + 128),
           dict(K={"bf16": 260, "fp8": 264}.get(fmt, 192)), dict(pairs=-1), dict(pairs=1 << 26, rows=1 << 26), dict(gated=2),
           dict(gated=1, N=63), dict(N=2 ** 31 - 1, os=2 ** 31 - 1, pairs=1 << 20),
           dict(N=1 << 20, os=1 << 20, pairs=1 << 22, rows=1 << 22)]
    bad += [dict(meta=None), dict(meta=A + (2 if fmt == "fp8" else 1))] if fmt != "bf16" else []
    bad += [dict(zeros=None)] if fmt == "int4_zp" else []
    bad += [dict(bias=A + 1)] if fmt != "int4" else []
    for b in bad:
        assert experts(gemv_lib, fmt, **b) == -2, b
    assert experts(gemv_lib, fmt, pairs=0, rows=0) == 0


def test_meta_shapes():
    from paia_gemv import ops
    ops.load()
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    i = lambda *s: e(*s, dtype=torch.int32)  # noqa: E731
    for x, res, dtype in ((e(5, 64), e(5, 64), torch.bfloat16), (e(5, 3, 64), e(5, 64, dtype=torch.float32), torch.float32),
                          (e(5, 64), None, torch.bfloat16)):
        h, r = ops.add_norm(x, res, e(64), weights=e(5, 3, dtype=torch.float32) if x.dim() == 3 else None)
        assert h.shape == r.shape == (5, 64) and h.dtype == torch.bfloat16 and r.dtype == dtype
    ids, w, o, f = ops.route_experts(e(7, 20), 3)
    assert ids.shape == w.shape == (7, 3) and o.shape == (21,) and f.shape == (21,)
    assert (ids.dtype, w.dtype, o.dtype, f.dtype) == (torch.int32, torch.float32, torch.int32, torch.int32)
    o, f = ops.expert_order(i(7, 3), 20)
    assert o.shape == (21,) and f.shape == (21,)
    x = e(7, 256)
    u8 = lambda *s: e(*s, dtype=torch.uint8)  # noqa: E731
    f32 = lambda *s: e(*s, dtype=torch.float32)  # noqa: E731
    for call, W in ((ops.experts_bf16, (e(20, 64, 256),)), (ops.experts_fp8, (u8(20, 64, 256), f32(20, 64))),
                    (ops.experts_int4, (u8(20, 64, 128), e(20, 64, 2, dtype=torch.float16))),
                    (ops.experts_int4_zp, (u8(20, 64, 128), e(20, 64, 2), u8(20, 64, 1)))):
        assert call(*W, x, o, f).shape == (21, 64) and call(*W, x, o, f, gated=True).shape == (21, 32)
        assert call(*W, x, o, f).dtype == torch.bfloat16
    assert ops.route_experts_workspace(100, 64, 4) > 0


def test_the_last_arguments_reach_the_abi(gemv_lib):
    """The loader's argument lists have the header's lengths."""
    lib = gemv_lib._lib
    for name, n in (("paia_add_norm", 22), ("paia_route_experts", 17), ("paia_expert_order", 9), ("paia_experts_bf16", 15),
                    ("paia_experts_fp8", 16), ("paia_experts_int4", 15), ("paia_experts_int4_zp", 17)):
        assert len(getattr(lib, name).argtypes) == n
    assert ctypes.sizeof(ctypes.c_longlong) == 8
