"""ops.paged_attention and GemvLib.paged_attention against the definition in 64 bits.

Tolerances. With A = sum of weight |v| and Q = the largest sum of |q_i k_i| |scale| of a token and head:
  a score is off by at most e = (D + 16) 2^-24 Q (fp32 products and sums of bf16 values, factor, exponent's argument);
  out: weights off by 2 e + 2^-20 (exponentials and the joins' factors), each rounded to bf16 (2^-8), sums of n terms
       (n/32 + 64) 2^-24, one rounding to bf16:  |out - ref| <= (2 e + 2^-20 + 2^-8 + (n/32 + 64) 2^-24) A + 2^-8 |ref|;
  lse: e + 2^-20 + (n/32 + 64) 2^-24 + 2^-22 |lse|.
"""
import math

import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, attention64, bits, make_cache, on
from gpu_util import note
from paia_gemv import load_lib, ops
from paia_gemv.loader import KVCache

pytestmark = pytest.mark.gpu


def operands(lens, T, heads, kv_heads, dim, fp8, layout, page, seed=1, sharp=1.0, extra=2):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width, pages = max(need + [1]) + extra, sum(need) + 3
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    order = torch.randperm(pages, generator=g).int()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    o = {"q": (torch.randn(len(lens), T, heads, dim, generator=g) * sharp).to(torch.bfloat16), "table": table,
         "k_cache": make_cache(pages, kv_heads, page, dim, fp8, layout, g),
         "v_cache": make_cache(pages, kv_heads, page, dim, fp8, layout, g),
         "lens": torch.tensor(lens, dtype=torch.int32), "k_scale": None, "v_scale": None}
    if fp8:
        o["k_scale"], o["v_scale"] = (torch.rand(2, kv_heads, generator=g) * 0.05 + 0.04).unbind()
    return o


def call(o, dev, **more):
    d = {k: on(v, dev) for k, v in o.items()}
    out, lse = ops.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["lens"], k_scale=d["k_scale"],
                                   v_scale=d["v_scale"], return_lse=True, **more)
    torch.cuda.synchronize()
    return out, lse


def check(o, out, lse, **more):
    ref, rlse, A, Q = attention64(o["q"], o["k_cache"], o["v_cache"], o["table"], o["lens"], k_scale=o["k_scale"],
                                  v_scale=o["v_scale"], **more)
    n, D = int(o["lens"].max()), o["q"].shape[-1]
    e = (D + 16) * F32_EPS * Q
    joins = 2.0 ** -20 + (n / 32 + 64) * F32_EPS
    out, lse = out.cpu().double().view(ref.shape), lse.cpu().double().view(rlse.shape)
    empty = rlse == -math.inf
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
    bound = (2 * e[..., None] + joins + BF16_HALF) * A + BF16_HALF * ref.abs()
    worst = ((out - ref).abs() - bound).max()
    assert worst <= 0, f"out beyond its bound by {worst:.3e}"
    off = ((lse - rlse).abs() - (e + joins + 2.0 ** -22 * rlse.abs()))[~empty]
    assert off.numel() == 0 or off.max() <= 0, f"lse beyond its bound by {off.max():.3e}"


LENS = [[1], [0], [31, 32, 33, 0, 1], [255, 257, 5, 300], [1000], [2049, 7, 513]]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layout,page", [("hpd", 16), ("phd", 24), ("gap", 1), ("hpd", 5), ("phd", 64), ("hpd", 300)])
def test_lengths_pages_layouts(cuda, dim, fp8, layout, page):
    for i, lens in enumerate(LENS):
        heads, kv_heads = [(8, 2), (7, 1), (3, 3), (32, 2)][i % 4]
        note(f"attention dim={dim} fp8={fp8} {layout} page={page} lens={lens} heads={heads}/{kv_heads}")
        o = operands(lens, 1, heads, kv_heads, dim, fp8, layout, page, seed=i)
        check(o, *call(o, cuda))


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (8, 8), (16, 1), (40, 2), (71, 1), (17, 17)])
def test_head_groups(cuda, heads, kv_heads):
    """Groups below, at and above the 16 columns that a block takes."""
    for fp8 in (False, True):
        note(f"attention groups {heads}/{kv_heads} fp8={fp8}")
        o = operands([700, 33], 1, heads, kv_heads, 128, fp8, "hpd", 16, seed=heads)
        check(o, *call(o, cuda))


@pytest.mark.parametrize("T", [2, 3, 5, 16])
@pytest.mark.parametrize("window", [0, 1, 2, 31, 100, 5000])
def test_several_tokens_and_windows(cuda, T, window):
    for lens, page, dim, fp8 in (([1, 2, 40, 0], 16, 128, False), ([1025, 64, 330], 8, 64, True),
                                 ([288, T, T - 1], 3, 128, False)):
        for heads, kv_heads in ((8, 2), (5, 1)):
            note(f"attention T={T} window={window} lens={lens} page={page} dim={dim} fp8={fp8} heads={heads}/{kv_heads}")
            o = operands(lens, T, heads, kv_heads, dim, fp8, "hpd", page, seed=T)
            check(o, *call(o, cuda, window=window), window=window)


def test_one_token_windows(cuda):
    for window in (1, 7, 32, 33, 500, 2 ** 31 - 1):
        note(f"attention window={window}")
        o = operands([900, 32, 64, 1, 501], 1, 8, 2, 128, False, "phd", 16, seed=window % 1000)
        check(o, *call(o, cuda, window=window), window=window)


@pytest.mark.parametrize("page", [16, 6])
def test_pages_outside_the_cache_hold_nothing(cuda, page):
    for T in (1, 3):
        note(f"attention holes page={page} T={T}")
        o = operands([400, 90, 33], T, 8, 2, 128, False, "hpd", page, seed=page)
        o["table"][0, 3:9] = -1
        o["table"][0, 0] = o["k_cache"].shape[0]
        o["table"][1] = -7
        o["table"][2, 0] = 2 ** 31 - 1
        check(o, *call(o, cuda))


def test_a_three_dimensional_query_and_lengths_beyond_the_table(cuda):
    o = operands([64, 40], 1, 8, 2, 64, False, "hpd", 16, extra=0)
    d = {k: on(v, cuda) for k, v in o.items()}
    out, lse = ops.paged_attention(d["q"][:, 0], d["k_cache"], d["v_cache"], d["table"], d["lens"] + 0, return_lse=True)
    assert out.shape == (2, 8, 64) and lse.shape == (2, 8)
    check(o, out, lse)
    far = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32)
    out, lse = ops.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["table"], far.to(cuda), return_lse=True)
    check({**o, "lens": far.clamp(max=64)}, out, lse)


@pytest.mark.parametrize("scale", [1.0, 0.0, -0.3, 4.0])
def test_scales(cuda, scale):
    o = operands([300], 1, 8, 2, 128, False, "hpd", 16, sharp=0.5)
    check(o, *call(o, cuda, scale=scale), scale=scale)


def test_peaked_scores(cuda):
    """Scores in the hundreds, so that nearly all the weight lies on one position and the running maximum keeps moving."""
    o = operands([1500, 600], 1, 8, 2, 128, False, "hpd", 16, sharp=40.0)
    check(o, *call(o, cuda))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("page", [16, 7])
def test_what_a_token_does_not_see_may_hold_anything(cuda, bad, page):
    """Bytes past the end of the last page, pages outside the sequence, positions before the window and, for earlier tokens
    of a draft, the later tokens' own rows: NaN and infinities there change nothing."""
    T, window, n = 3, 70, 203
    o = operands([n, 50], T, 8, 2, 128, False, "hpd", page, seed=5)
    want = call(o, cuda, window=window)
    check(o, *want, window=window)
    seen = torch.zeros(o["k_cache"].shape[0], page, dtype=torch.bool)
    for b, m in enumerate(o["lens"].tolist()):
        for p in range(max(0, m - (T - 1) - window), m):
            seen[int(o["table"][b, p // page]), p % page] = True
    k, v = o["k_cache"].clone(), o["v_cache"].clone()
    for c in (k, v):
        c.transpose(1, 2)[~seen] = bad
    note(f"attention unseen {bad} page={page}")
    got = call({**o, "k_cache": k, "v_cache": v}, cuda, window=window)
    assert torch.equal(bits(got[0]), bits(want[0])) and torch.equal(got[1], want[1])
    # the last token's row is seen by the last token alone
    p = n - 1
    for c in (k, v):
        c[int(o["table"][0, p // page]), :, p % page] = bad
    note(f"attention last row {bad} page={page}")
    got = call({**o, "k_cache": k, "v_cache": v}, cuda, window=window)
    assert torch.equal(bits(got[0][:, :T - 1]), bits(want[0][:, :T - 1])) and torch.equal(got[1][:, :T - 1], want[1][:, :T - 1])
    assert torch.equal(bits(got[0][1]), bits(want[0][1]))
    assert not got[0][0, T - 1].isfinite().all()


def test_a_nan_that_is_seen(cuda):
    o = operands([500, 500], 1, 8, 2, 128, False, "hpd", 16, seed=6)
    o["k_cache"][int(o["table"][0, 3]), 1, 2, 5] = float("nan")
    out, lse = call(o, cuda)
    assert out[0, 0, 4:].isnan().all() and lse[0, 0, 4:].isnan().all()
    assert out[0, 0, :4].isfinite().all() and out[1].isfinite().all() and lse[1].isfinite().all()


def test_many_sequences(cuda):
    """More sequences than lanes of a wave, and more than the pieces that are aimed at."""
    g = torch.Generator().manual_seed(3)
    for B in (65, 700):
        lens = torch.randint(0, 90, (B,), generator=g).tolist()
        lens[B // 2] = 3001
        note(f"attention B={B}")
        o = operands(lens, 1, 4, 2, 64, False, "hpd", 16, seed=B)
        check(o, *call(o, cuda))


def test_offsets_beyond_32_bits(cuda):
    """Pages at the end of caches of 6 GiB give what the same pages give in a small cache, bit for bit."""
    for fp8 in (False, True):
        o = operands([330, 1000], 1, 16, 8, 128, fp8, "hpd", 16, seed=2)
        want = call(o, cuda)
        d = {k: on(v, cuda) for k, v in o.items()}
        n = d["k_cache"].shape[0]
        pages = 6 * 2 ** 30 // (8 * 16 * 128 * d["k_cache"].element_size())
        big = []
        for c in (d["k_cache"], d["v_cache"]):
            b = torch.empty(pages, 8, 16, 128, dtype=c.dtype, device=cuda)
            raw = torch.uint8 if fp8 else c.dtype
            b.view(raw)[pages - n:] = c.view(raw)
            big.append(b)
        table = torch.where(d["table"] >= 0, d["table"] + (pages - n), d["table"]).int()
        note(f"attention far pages fp8={fp8}")
        got = ops.paged_attention(d["q"], *big, table, d["lens"], k_scale=d["k_scale"], v_scale=d["v_scale"],
                                  return_lse=True)
        assert torch.equal(bits(got[0]), bits(want[0])) and torch.equal(got[1], want[1])
        del big, b


def test_strided_query_out_and_workspace(cuda):
    """q as a view of a fused projection, a caller's output and workspace: the same bits, also in a workspace of NaN."""
    o = operands([2000, 90], 1, 8, 2, 128, False, "hpd", 16, seed=4)
    want, _ = call(o, cuda)
    d = {k: on(v, cuda) for k, v in o.items()}
    wide = torch.full((2, 12 * 128), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, :1024] = d["q"].view(2, 1024)
    need = ops.paged_attention_workspace(d["k_cache"], d["table"].shape[1], 2, 1, 8)
    assert need > 0
    space = torch.full((need // 4,), float("nan"), device=cuda)
    out = torch.full((2, 8, 128), float("nan"), dtype=torch.bfloat16, device=cuda)
    r = ops.paged_attention(wide[:, :1024].unflatten(1, (8, 128)), d["k_cache"], d["v_cache"], d["table"], d["lens"],
                            out=out, workspace=space)
    assert r is out and torch.equal(bits(out).view(-1), bits(want).view(-1))


def test_graph_follows_the_lengths(cuda):
    """One captured call replayed as the sequences grow, eager work between the replays."""
    o = operands([3000, 2500], 1, 8, 2, 128, False, "hpd", 16, seed=8)
    d = {k: on(v, cuda) for k, v in o.items()}
    lens = torch.tensor([1, 1], dtype=torch.int32, device=cuda)
    call_it = lambda: ops.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["table"], lens, return_lse=True)  # noqa: E731
    call_it()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call_it()
    for a in (1, 40, 700, 2500, 3):
        lens.copy_(torch.tensor([min(3000, a + 9), a]))
        junk = torch.randn(1 << 20, device=cuda).mul_(2.0)
        torch.cuda.synchronize()
        note(f"attention replay at {a}")
        graph.replay()
        torch.cuda.synchronize()
        want = call_it()
        assert torch.equal(bits(out), bits(want[0])) and torch.equal(lse, want[1]), a
        del junk


def test_c_abi_and_another_stream(cuda):
    o = operands([1200, 77], 2, 28, 4, 128, True, "hpd", 16, seed=9)
    want, wlse = call(o, cuda, window=300)
    d = {k: on(v, cuda) for k, v in o.items()}
    lib = load_lib()
    cache = KVCache(d["k_cache"].data_ptr(), d["v_cache"].data_ptr(), d["k_cache"].shape[0], 16, 4, 128, True,
                    d["k_scale"].data_ptr(), d["v_scale"].data_ptr())
    width = d["table"].shape[1]
    need = lib.paged_attention_workspace(cache, width, 2, 2, 28)
    assert need == ops.paged_attention_workspace(d["k_cache"], width, 2, 2, 28)
    out, lse = torch.empty_like(d["q"]), torch.empty(2, 2, 28, device=cuda)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        space = torch.empty(max(need, 16), dtype=torch.uint8, device=cuda)
        q = (d["q"].float() * 2.0).to(torch.bfloat16).div_(2.0)
        lib.paged_attention(q.data_ptr(), cache, d["table"].data_ptr(), width, d["lens"].data_ptr(), out.data_ptr(), 2, 2,
                            28, 128 ** -0.5, 300, lse.data_ptr(), space.data_ptr(), need)
    st.synchronize()
    assert torch.equal(bits(out), bits(want)) and torch.equal(lse, wlse)


def test_no_sequences(cuda):
    o = operands([40], 1, 8, 2, 128, False, "hpd", 16)
    d = {k: on(v, cuda) for k, v in o.items()}
    out = ops.paged_attention(d["q"][:0], d["k_cache"], d["v_cache"], d["table"][:0], d["lens"][:0])
    assert out.shape == (0, 1, 8, 128)


def test_refusals(cuda):
    o = operands([40, 50], 1, 8, 2, 128, False, "hpd", 16)
    d = {k: on(v, cuda) for k, v in o.items()}

    def refused(match, error=RuntimeError, **change):
        a = {**d, "window": 0, "out": None, "workspace": None, "return_lse": False, **change}
        with pytest.raises(error, match=match):
            ops.paged_attention(a["q"], a["k_cache"], a["v_cache"], a["table"], a["lens"], window=a["window"],
                                k_scale=a["k_scale"], v_scale=a["v_scale"], out=a["out"], workspace=a["workspace"],
                                return_lse=a["return_lse"])

    refused("bfloat16", q=d["q"].half())
    refused("head_dim", q=d["q"][..., :64].contiguous())
    refused("multiple", q=d["q"][:, :, :7])
    refused("last dimension", q=d["q"].transpose(2, 3).contiguous().transpose(2, 3))
    refused("lens", lens=d["lens"].long())
    refused("lens", lens=d["lens"][:1])
    refused("lens must be on", lens=d["lens"].cpu())
    refused("block_table", table=d["table"].long())
    refused("block_table", table=d["table"][:1])
    refused("window", window=-1)
    refused("out must", out=torch.empty(2, 8, 127, dtype=torch.bfloat16, device=cuda))
    refused("return_lse", error=ValueError, out=torch.empty_like(d["q"]), return_lse=True)
    refused("e4m3 cache", v_scale=torch.ones(2, device=cuda))
    refused("both", k_cache=d["k_cache"].view(torch.int16))
    big = operands([4000], 1, 8, 2, 128, False, "hpd", 16)
    b = {k: on(v, cuda) for k, v in big.items()}
    refused("workspace", q=b["q"], k_cache=b["k_cache"], v_cache=b["v_cache"], table=b["table"], lens=b["lens"],
            workspace=torch.empty(64, device=cuda))
    odd = torch.empty(2, 8 * 128 + 4, dtype=torch.bfloat16, device=cuda)
    refused("-2", q=odd[:, :1024].unflatten(1, (8, 128)))


@pytest.mark.parametrize("dim,fp8,page", [(64, False, 16), (64, True, 7), (128, False, 16), (128, False, 9), (128, True, 16)])
def test_column_tiles_together(cuda, dim, fp8, page):
    """Tables wide enough for the forms whose blocks take two or three tiles of columns (and those that never do): the same
    sequences in a narrow and a wide table, with drafts, a window, holes and values nobody sees."""
    wide = -(-(300 << 20) // (2 * 2 * 2 * dim * (1 if fp8 else 2) * page))
    for T, heads, window in ((5, 8, 0), (5, 16, 0), (3, 40, 100), (1, 70, 0)):
        note(f"attention column tiles dim={dim} fp8={fp8} page={page} T={T} heads={heads} window={window}")
        o = operands([700, 37], T, heads, 2, dim, fp8, "phd", page, seed=T + heads)
        o["table"][0, 2] = -1
        narrow = call(o, cuda, window=window)
        check(o, *narrow, window=window)
        table = torch.full((2, wide), -1, dtype=torch.int32)
        table[:, :o["table"].shape[1]] = o["table"]
        got = call({**o, "table": table}, cuda, window=window)
        check(o, *got, window=window)
        if T > 1:      # the last row of a sequence, which only its last token sees
            p = 699
            for c in ("k_cache", "v_cache"):
                o[c] = o[c].clone()
                o[c][int(o["table"][0, p // page]), :, p % page] = float("nan")
            bad = call({**o, "table": table}, cuda, window=window)
            assert torch.equal(bits(bad[0][:, :T - 1]), bits(got[0][:, :T - 1])) and torch.equal(bad[1][:, :T - 1], got[1][:, :T - 1])
            assert bad[0][0, T - 1].isnan().all() and torch.equal(bits(bad[0][1]), bits(got[0][1]))
