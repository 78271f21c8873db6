"""paged_attention's weights enter their product with V as two bf16 terms. A bound that sees it when one of them is lost.

As test_gpu_attention.py derives it, with A = sum of weight |v|, Q = the largest sum of |q_i k_i| |scale|, e = (D + 16) 2^-24 Q, but
2^-16 for the weights' rounding: the first term of a weight in [1, 2) is cut at 2^-7, the second keeps 8 bits of what is left, so half
of 2^-15 is lost at most, and less where the first is rounded:
  |out - ref| <= (2 e + 2^-20 + 2^-16 + (n/32 + 64) 2^-24) A + 2^-8 |ref|.
"""
import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, attention64, codes, make_cache, on

CASES = [(5, 256), (33, 64), (33, 128), (33, 256), (300, 128), (700, 64), (700, 128), (2049, 64)]


def operands(n, D, fp8, T=1, heads=8, page=16):
    """Queries a quarter of the usual size: the bound's part for the scores is then small beside that for the weights."""
    g = torch.Generator().manual_seed(n + D)
    pages = -(-n // page)
    o = {"q": (torch.randn(1, T, heads, D, generator=g) * 0.25).to(torch.bfloat16),
         "k_cache": make_cache(pages, 2, page, D, fp8, "hpd", g), "v_cache": make_cache(pages, 2, page, D, fp8, "hpd", g),
         "table": torch.randperm(pages, generator=g).int()[None], "lens": torch.tensor([n], dtype=torch.int32)}
    s = torch.full((2,), 0.0625) if fp8 else None
    return o, s


def bound(o, s):
    ref, _, A, Q = attention64(o["q"], o["k_cache"], o["v_cache"], o["table"], o["lens"], k_scale=s, v_scale=s)
    n, D = int(o["lens"][0]), o["q"].shape[-1]
    e = (D + 16) * F32_EPS * Q
    return ref, (2 * e[..., None] + 2.0 ** -20 + 2.0 ** -16 + (n / 32 + 64) * F32_EPS) * A + BF16_HALF * ref.abs()


def rounded(o, s, terms):
    """The definition in 64 bits with the weights in one bf16 term (the nearest) or two (cut, and the rest's nearest)."""
    q, n = o["q"][0, 0].double(), int(o["lens"][0])
    H, D = o["k_cache"].shape[1], q.shape[-1]
    k, v = (codes(o[c][o["table"][0].long()]).transpose(0, 1).reshape(H, -1, D)[:, :n] * (1.0 if s is None else float(s[0]))
            for c in ("k_cache", "v_cache"))
    a = torch.matmul(q.view(H, -1, D), k.transpose(1, 2)) * D ** -0.5
    w = torch.exp(a - a.amax(-1, keepdim=True))
    if terms == 1:
        p = w.to(torch.bfloat16).double()
    else:
        top = (w.float().view(torch.int32) & -65536).view(torch.float32).double()
        p = top + (w - top).to(torch.bfloat16).double()
    return (torch.matmul(p, v) / w.sum(-1, keepdim=True)).to(torch.bfloat16).double().view(1, 1, -1, D)


@pytest.mark.parametrize("n,D", CASES)
@pytest.mark.parametrize("fp8", [False, True])
def test_the_bound_tells_one_term_from_two(n, D, fp8):
    o, s = operands(n, D, fp8)
    ref, limit = bound(o, s)
    assert ((rounded(o, s, 2) - ref).abs() <= limit).all()
    assert ((rounded(o, s, 1) - ref).abs() > 2.0 * limit).any()


@pytest.mark.gpu
@pytest.mark.parametrize("n,D", CASES)
@pytest.mark.parametrize("fp8", [False, True])
def test_weights_keep_sixteen_bits(cuda, n, D, fp8):
    """Also where tokens of a draft take different tiles, and where a block takes several tiles of columns (a wide table)."""
    from gpu_util import note
    from paia_gemv import ops
    wide = -(-(300 << 20) // (2 * 2 * D * (1 if fp8 else 2) * 16))
    for T, heads, width in ((1, 8, None), (3, 8, None), (3, 24, wide)):
        note(f"attention precision n={n} D={D} fp8={fp8} T={T} heads={heads} width={width}")
        o, s = operands(n, D, fp8, T, heads)
        ref, limit = bound(o, s)
        table = o["table"]
        if width is not None:
            table = torch.cat([table, torch.full((1, width), -1, dtype=torch.int32)], dim=1)
        d = [on(t, cuda) for t in (o["q"], o["k_cache"], o["v_cache"], table, o["lens"], s)]
        out = ops.paged_attention(*d[:5], k_scale=d[5], v_scale=d[5])
        worst = ((out.cpu().double() - ref).abs() / limit).max()
        assert worst <= 1.0, f"{worst:.3f} of the bound"
