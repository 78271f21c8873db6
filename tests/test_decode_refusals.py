"""Host-side checks of the entry points between and beside the projections: every call below returns from them, nothing is
launched (no GPU needed)."""
import ctypes

import pytest
import torch

from paia_gemv.loader import KVCache

A = 1 << 20      # a 16-byte-aligned address, never dereferenced


def cache(**change):
    c = KVCache(A, A, 10, 16, 8, 128, change.pop("fp8", False))
    for k, v in change.items():
        if k in ("k_strides", "v_strides"):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


BAD_CACHES = [dict(k=None), dict(v=A + 8), dict(pages=0), dict(page_size=0), dict(kv_heads=0), dict(head_dim=96),
              dict(fp8=2), dict(k_scale=A + 2), dict(k_strides=(16384, 2048, 132)), dict(v_strides=(-16384, 2048, 128)),
              dict(fp8=True, v_strides=(16384, 2048, 136))]


def rope(lib, c, **change):
    a = dict(qkv=A, stride=48 * 128, positions=A, cos_sin=A, context=100, rotary=128, q_norm=None, k_norm=None, slots=A,
             q=A + 4096, M=4, heads=32)
    a.update(change)
    return lib._lib.paia_rope_append(a["qkv"], a["stride"], a["positions"], a["cos_sin"], a["context"], a["rotary"], 0,
                                     a["q_norm"], a["k_norm"], 1e-6, a["slots"], ctypes.byref(c) if c else None, a["q"],
                                     a["M"], a["heads"], None)


def test_rope_append_refusals(gemv_lib):
    for bad in BAD_CACHES:
        assert rope(gemv_lib, cache(**bad)) == -2, bad
    assert rope(gemv_lib, None) == -2
    for bad in (dict(qkv=A + 8), dict(qkv=None), dict(stride=6148), dict(positions=A + 4), dict(cos_sin=A + 4),
                dict(context=0), dict(rotary=0), dict(rotary=136), dict(rotary=144), dict(rotary=24), dict(q_norm=A + 8),
                dict(k_norm=A + 2), dict(slots=None), dict(q=A + 4), dict(q=A), dict(M=-1), dict(heads=0)):
        assert rope(gemv_lib, cache(), **bad) == -2, bad
    assert rope(gemv_lib, cache(), M=0) == 0


def test_rope_append_meta_shape():
    from paia_gemv import ops
    ops.load()
    m = torch.device("meta")
    kc = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16, device=m)
    q = torch.ops.paia_gemv.rope_append(torch.empty(3, 8 * 64, dtype=torch.bfloat16, device=m), torch.empty(3, device=m),
                                        torch.empty(9, 64, device=m), kc, kc.clone(), torch.empty(3, device=m), 4)
    assert q.shape == (3, 4, 64) and q.dtype == torch.bfloat16


def test_rope_table():
    from paia_gemv import ops
    t = ops.rope_table(50, 16, base=100.0)
    assert t.shape == (50, 16) and t.dtype == torch.float32
    f = 100.0 ** (-2.0 * 3 / 16)
    assert abs(float(t[37, 3]) - float(torch.tensor(37 * f, dtype=torch.float64).cos())) <= 2.0 ** -24
    assert abs(float(t[37, 8 + 3]) - float(torch.tensor(37 * f, dtype=torch.float64).sin())) <= 2.0 ** -24
    assert torch.equal(ops.rope_table(50, 16, inverse_frequencies=[0.5] * 8)[2, :8], torch.full((8,), 1.0, dtype=torch.float64).cos().float())


@pytest.mark.parametrize("bad", [dict(context=-5, rotary=16)])
def test_rope_table_refuses(bad):
    from paia_gemv import ops
    with pytest.raises(RuntimeError):
        ops.rope_table(**bad)


def attention(lib, c, **change):
    a = dict(q=A, strides=(4096, 4096, 128), table=A, stride=64, width=64, lens=A, window=0, out=A + 4096, lse=None, B=2, T=1,
             heads=32, space=A, bytes=1 << 40)
    a.update(change)
    st = (ctypes.c_longlong * 3)(*a["strides"]) if a["strides"] else None
    return lib._lib.paia_paged_attention(a["q"], st, ctypes.byref(c) if c else None, a["table"], a["stride"], a["width"],
                                         a["lens"], 0.1, a["window"], a["out"], a["lse"], a["B"], a["T"], a["heads"],
                                         a["space"], a["bytes"], None)


def test_paged_attention_refusals(gemv_lib):
    for bad in BAD_CACHES:
        assert attention(gemv_lib, cache(**bad)) == -2, bad
    assert attention(gemv_lib, None) == -2
    for bad in (dict(q=None), dict(q=A + 8), dict(strides=None), dict(strides=(4096, 4096, 132)),
                dict(strides=(-4096, 4096, 128)), dict(table=None), dict(table=A + 2), dict(stride=-1), dict(width=-1),
                dict(lens=None), dict(lens=A + 1), dict(window=-1), dict(out=None), dict(out=A + 8), dict(out=A), dict(lse=A + 2),
                dict(B=-1), dict(T=0), dict(heads=0), dict(heads=30), dict(space=None), dict(space=A + 8), dict(bytes=100),
                dict(T=1 << 30), dict(B=1 << 28)):
        assert attention(gemv_lib, cache(), **bad) == -2, bad
    assert attention(gemv_lib, cache(), B=0) == 0


def test_paged_attention_workspace(gemv_lib):
    need = lambda w, B=2, T=1, heads=32, **c: gemv_lib._lib.paia_paged_attention_workspace(  # noqa: E731
        ctypes.byref(cache(**c)), w, B, T, heads)
    assert need(0) == 0 and need(1) == 0                 # sequences of one piece are not joined
    assert 0 < need(1000) <= need(8192) and need(8192) == need(100000)   # bounded by the chip, not by the length
    assert need(100, heads=30) == -2 and need(-1) == -2 and need(100, T=0) == -2 and need(100, page_size=0) == -2
    assert need(2 ** 31 - 1, page_size=2 ** 31 - 1) > 0
    assert gemv_lib.paged_attention_workspace(cache(), 1000, 2, 1, 32) == need(1000)
    with pytest.raises(RuntimeError, match="-2"):
        gemv_lib.paged_attention_workspace(cache(), 1000, 2, 1, 30)


def test_paged_attention_meta_shapes():
    from paia_gemv import ops
    ops.load()
    m = torch.device("meta")
    kc = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16, device=m)
    q = torch.empty(3, 4, 8, 64, dtype=torch.bfloat16, device=m)
    table, lens = torch.empty(3, 5, dtype=torch.int32, device=m), torch.empty(3, dtype=torch.int32, device=m)
    assert torch.ops.paia_gemv.paged_attention(q, kc, kc, table, lens).shape == q.shape
    out, lse = torch.ops.paia_gemv.paged_attention_lse(q, kc, kc, table, lens)
    assert out.shape == q.shape and lse.shape == (3, 4, 8) and lse.dtype == torch.float32


def lora(lib, splits=(64, 32), **change):
    a = dict(y=A, ys=96, x=A, xs=128, A=A, B=A, ids=A, scaling=None, out=A, os=96, M=4, K=128, rank=40, adapters=3, space=A,
             bytes=1 << 40, slices=len(splits) if splits else 1)
    a.update(change)
    sp = (ctypes.c_int * len(splits))(*splits) if splits else None
    return lib._lib.paia_lora_add(a["y"], a["ys"], a["x"], a["xs"], a["A"], a["B"], a["ids"], a["scaling"], a["out"],
                                  a["os"], a["M"], a["K"], a["rank"], sp, a["slices"], a["adapters"], a["space"],
                                  a["bytes"], None)


def test_lora_add_refusals(gemv_lib):
    for bad in (dict(y=None), dict(y=A + 1), dict(ys=-1), dict(x=A + 8), dict(xs=100), dict(xs=-128), dict(A=None),
                dict(A=A + 4), dict(B=A + 2), dict(ids=None), dict(ids=A + 2), dict(scaling=A + 2), dict(out=None),
                dict(out=A + 1), dict(os=95), dict(M=-1), dict(K=0), dict(K=100), dict(rank=0), dict(rank=12),
                dict(rank=264), dict(adapters=0), dict(slices=0), dict(slices=9, splits=(1,) * 9), dict(splits=None),
                dict(splits=(64, 0)), dict(splits=(64, -1)), dict(splits=(2 ** 31 - 1, 2 ** 31 - 1)), dict(space=None),
                dict(space=A + 4), dict(bytes=64)):
        assert lora(gemv_lib, **bad) == -2, bad
    assert lora(gemv_lib, M=0) == 0
    need = gemv_lib.lora_add_workspace
    assert need(1000, 512, 40, [64, 32]) == need(256, 512, 40, [64, 32]) > need(4, 512, 40, [64, 32]) > 0
    assert need(1, 4096, 16, [4096, 1024, 1024]) == 0            # one launch, nothing kept
    for bad in ((4, 512, 12, [64]), (4, 512, 16, [64] * 9), (-1, 512, 16, [64]), (4, 100, 16, [64]), (4, 512, 16, [64, 0])):
        with pytest.raises(RuntimeError, match="-2"):
            need(*bad)


def test_lora_add_meta_shape():
    from paia_gemv import ops
    ops.load()
    e = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="meta")  # noqa: E731
    out = torch.ops.paia_gemv.lora_add(e(3, 40), e(3, 64), e(2, 8, 64), e(2, 40, 8), torch.empty(3, device="meta"))
    assert out.shape == (3, 40) and out.dtype == torch.bfloat16
