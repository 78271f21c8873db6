"""ops.rope_append and GemvLib.rope_append against the definition in 64 bits.

Tolerances: every output is fp32 arithmetic rounded once. The norm and the rotation are fewer than 300 fp32 operations, in
absolute terms within 64 * 2^-24 of the head's largest term (the sum of squares adds positive terms); then one rounding to
bf16 (2^-8 of the value) or to e4m3 (2^-4 of the value, 2^-10 absolute among the subnormals), times the factor.
"""
import itertools

import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, bits, codes, make_cache, on, rope64
from gpu_util import note
from paia_gemv import load_lib, ops
from paia_gemv.loader import KVCache

pytestmark = pytest.mark.gpu


def operands(M, heads, kv_heads, dim, rot, fp8, layout, page, norm, seed=1, pages=None, context=4096):
    g = torch.Generator().manual_seed(seed)
    pages = pages or max(2, -(-2 * M // page))
    o = {"qkv": torch.randn(M, (heads + 2 * kv_heads) * dim, generator=g).to(torch.bfloat16),
         "positions": torch.randint(0, context, (M,), generator=g), "cos_sin": ops.rope_table(context, rot),
         "k_cache": make_cache(pages, kv_heads, page, dim, fp8, layout, g),
         "v_cache": make_cache(pages, kv_heads, page, dim, fp8, layout, g),
         "slots": torch.randperm(pages * page, generator=g)[:M]}
    w = lambda: (1.0 + 0.2 * torch.randn(dim, generator=g)).to(torch.bfloat16)  # noqa: E731
    o["q_norm"], o["k_norm"] = (w(), w()) if norm else (None, None)
    sc = lambda: torch.rand(kv_heads, generator=g) * 0.02 + 0.01  # noqa: E731
    o["k_scale"], o["v_scale"] = (sc(), sc()) if fp8 else (None, None)
    return o


def check(o, q, k_cache, v_cache, heads, kv_heads, dim, pairs, page):
    """q and the written slots within tolerance of the definition, everything else of the cache bit for bit as it was."""
    rq, rk, rv = rope64(o["qkv"], o["positions"], o["cos_sin"], heads, kv_heads, dim, o["q_norm"], o["k_norm"], 1e-6, pairs)
    slack = lambda r: 64 * F32_EPS * r.abs().amax(-1, keepdim=True)  # noqa: E731
    q = q.cpu().double().view(rq.shape)
    assert ((q - rq).abs() <= BF16_HALF * rq.abs() + slack(rq)).all(), "q"
    pages = k_cache.shape[0]
    keep = (o["slots"] >= 0) & (o["slots"] < pages * page)
    at = (o["slots"][keep] // page, slice(None), o["slots"][keep] % page)
    for name, cache, ref in (("k", k_cache, rk), ("v", v_cache, rv)):
        f = 1.0 if o[name + "_scale"] is None else o[name + "_scale"].double()[:, None]
        got, ref = codes(cache)[at] * f, ref[keep]
        if o[name + "_scale"] is None:
            assert ((got - ref).abs() <= BF16_HALF * ref.abs() + slack(ref)).all(), name
        else:
            lim = ref.clamp(min=-448.0 * f, max=448.0 * f)
            assert ((got - lim).abs() <= 2.0 ** -4 * lim.abs() + 2.0 ** -10 * f + slack(ref)).all(), name
        before, after = bits(o[name + "_cache"]).clone(), bits(cache).clone()
        before[at] = 0
        after[at] = 0
        assert torch.equal(before, after), f"{name}: something else was written"


def call(o, dev, heads, pairs=False, **more):
    d = {k: on(v, dev) for k, v in o.items()}
    q = ops.rope_append(d["qkv"], d["positions"], d["cos_sin"], d["k_cache"], d["v_cache"], d["slots"], heads,
                        q_norm=d["q_norm"], k_norm=d["k_norm"], interleaved=pairs, k_scale=d["k_scale"],
                        v_scale=d["v_scale"], **more)
    torch.cuda.synchronize()
    return q, d["k_cache"], d["v_cache"]


@pytest.mark.parametrize("dim,rots", [(64, (64, 48, 16)), (128, (128, 64, 112)), (256, (256, 16, 240))])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("pairs", [False, True])
def test_rope_append(cuda, dim, rots, fp8, pairs):
    heads_of = itertools.cycle([(32, 8), (7, 1), (28, 4), (3, 3), (1, 1)])
    for (M, layout, page), rot, norm in itertools.product([(1, "hpd", 16), (5, "phd", 24), (67, "gap", 1)], rots,
                                                          (False, True)):
        heads, kv_heads = next(heads_of)
        note(f"rope M={M} {layout} page={page} dim={dim} rot={rot} norm={norm} fp8={fp8} pairs={pairs} heads={heads}")
        o = operands(M, heads, kv_heads, dim, rot, fp8, layout, page, norm)
        o["slots"][M // 2] = [-1, 10 ** 12, o["slots"][M // 2]][M % 3]
        check(o, *call(o, cuda, heads, pairs), heads, kv_heads, dim, pairs, page)


@pytest.mark.parametrize("only", ["q_norm", "k_norm"])
def test_one_norm_alone(cuda, only):
    o = operands(4, 8, 2, 128, 128, False, "hpd", 16, True)
    o["k_norm" if only == "q_norm" else "q_norm"] = None
    check(o, *call(o, cuda, 8), 8, 2, 128, False, 16)


def test_no_tokens(cuda):
    o = operands(1, 8, 2, 128, 128, False, "hpd", 16, False)
    for n in ("qkv", "positions", "slots"):
        o[n] = o[n][:0]
    q, k, _ = call(o, cuda, 8)
    assert q.shape == (0, 8, 128) and torch.equal(bits(k), bits(o["k_cache"]))


def test_strided_rows_and_out(cuda):
    """qkv as the left part of a wider tensor, and a caller's output tensor."""
    o = operands(9, 4, 2, 64, 64, False, "phd", 16, True)
    want = call(o, cuda, 4)
    wide = torch.full((9, 8 * 64 + 24), float("nan"), dtype=torch.bfloat16)
    wide[:, :512] = o["qkv"]
    wide = wide.to(cuda)
    d = {k: on(v, cuda) for k, v in o.items()}
    out = torch.full((9, 4, 64), float("nan"), dtype=torch.bfloat16, device=cuda)
    r = ops.rope_append(wide[:, :512], d["positions"], d["cos_sin"], d["k_cache"], d["v_cache"], d["slots"], 4,
                        q_norm=d["q_norm"], k_norm=d["k_norm"], out=out)
    torch.cuda.synchronize()
    assert r is out and torch.equal(bits(out), bits(want[0]))
    assert torch.equal(bits(d["k_cache"]), bits(want[1])) and torch.equal(bits(d["v_cache"]), bits(want[2]))


def test_positions_outside_the_table_give_nan(cuda):
    o = operands(3, 4, 2, 128, 64, False, "hpd", 16, False, context=100)
    o["positions"] = torch.tensor([-1, 50, 100])
    q, k, v = call(o, cuda, 4)
    q = q.cpu().float()
    assert q[[0, 2], :, :64].isnan().all() and q[[0, 2], :, 64:].isfinite().all() and q[1].isfinite().all()
    s = o["slots"]
    assert codes(k)[s // 16, :, s % 16][[0, 2], :, :64].isnan().all()
    assert torch.equal(codes(v)[s // 16, :, s % 16], o["qkv"].double().view(3, 8, 128)[:, 6:])


def test_not_finite_and_large_values(cuda):
    """NaN and infinities stay in their own head; e4m3 clamps to +-448 times the factor and keeps NaN."""
    for fp8 in (False, True):
        o = operands(2, 2, 2, 128, 128, fp8, "hpd", 16, False)
        x = o["qkv"].view(2, 6, 128)
        x[0, 2, 5], x[0, 4, 0], x[0, 4, 1], x[0, 4, 2] = float("nan"), float("inf"), float("-inf"), 3e38
        x[0, 4, 3], x[0, 5, 7] = float("nan"), -1e4
        q, k, v = call(o, cuda, 2)
        assert q.isfinite().all()
        s = o["slots"]
        k, v = codes(k)[s // 16, :, s % 16], codes(v)[s // 16, :, s % 16]
        assert k[0, 0, [5, 69]].isnan().all() and int(k.isnan().sum()) == 2
        want = [448.0, -448.0, 448.0] if fp8 else [float("inf"), float("-inf"), float(torch.tensor(3e38).bfloat16())]
        assert v[0, 0, :3].tolist() == want and v[0, 0, 3].isnan() and int(v.isnan().sum()) == 1
        assert v[0, 1, 7] == (-448.0 if fp8 else float(torch.tensor(-1e4).bfloat16()))


def test_slots_beyond_32_bits(cuda):
    """A cache of 6 GiB: the last page's offset needs more than 32 bits."""
    o = operands(2, 8, 8, 128, 128, False, "hpd", 16, False)
    d = {k: on(v, cuda) for k, v in o.items()}
    pages = 6 * 2 ** 30 // (8 * 16 * 128 * 2)
    k, v = (torch.empty(pages, 8, 16, 128, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    slots = torch.tensor([pages * 16 - 1, pages * 8 + 3])
    ops.rope_append(d["qkv"], d["positions"], d["cos_sin"], k, v, slots.to(cuda), 8)
    small = call(o, cuda, 8)
    for big, ref in ((k, small[1]), (v, small[2])):
        got = big[slots.to(cuda) // 16, :, slots.to(cuda) % 16]
        assert torch.equal(bits(got), bits(ref.cpu()[o["slots"] // 16, :, o["slots"] % 16]))


def test_c_abi_and_another_stream(cuda):
    """GemvLib.rope_append with addresses, on a stream of its own behind work of that stream, equals the torch op."""
    o = operands(6, 28, 4, 128, 128, True, "hpd", 16, True)
    want = call(o, cuda, 28)
    d = {k: on(v, cuda) for k, v in o.items()}
    cache = KVCache(d["k_cache"].data_ptr(), d["v_cache"].data_ptr(), d["k_cache"].shape[0], 16, 4, 128, True,
                    d["k_scale"].data_ptr(), d["v_scale"].data_ptr())
    out = torch.empty(6, 28, 128, dtype=torch.bfloat16, device=cuda)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        qkv = (d["qkv"].float() * 2.0).to(torch.bfloat16).div_(2.0)
        load_lib().rope_append(qkv.data_ptr(), qkv.stride(0), d["positions"].data_ptr(), d["cos_sin"].data_ptr(), 4096,
                               128, d["slots"].data_ptr(), cache, out.data_ptr(), 6, 28, d["q_norm"].data_ptr(),
                               d["k_norm"].data_ptr())
    st.synchronize()
    assert torch.equal(bits(out), bits(want[0])) and torch.equal(bits(d["k_cache"]), bits(want[1]))
    assert torch.equal(bits(d["v_cache"]), bits(want[2]))


def test_refusals(cuda):
    o = operands(3, 4, 2, 128, 128, False, "hpd", 16, False)
    d = {k: on(v, cuda) for k, v in o.items()}

    def refused(match, heads=4, **change):
        a = {**d, **change}
        with pytest.raises(RuntimeError, match=match):
            ops.rope_append(a["qkv"], a["positions"], a["cos_sin"], a["k_cache"], a["v_cache"], a["slots"], heads,
                            q_norm=a["q_norm"], k_norm=a["k_norm"], k_scale=a["k_scale"], v_scale=a["v_scale"])

    refused("bfloat16", qkv=d["qkv"].float())
    refused("columns", heads=5)
    refused("num_heads", heads=0)
    refused("contiguous rows", qkv=d["qkv"].t().contiguous().t())
    refused("positions", positions=d["positions"].int())
    refused("positions", positions=d["positions"][:2])
    refused("slots", slots=d["slots"].cpu())
    refused("cos_sin", cos_sin=d["cos_sin"].double())
    refused("-2", cos_sin=d["cos_sin"][:, :120].contiguous())
    refused("both", v_cache=d["v_cache"].float())
    refused("both", v_cache=d["v_cache"][:1])
    refused("last dimension", k_cache=d["k_cache"].transpose(2, 3).contiguous().transpose(2, 3))
    refused("e4m3 cache", k_scale=torch.ones(2, device=cuda))
    refused("q_norm", q_norm=torch.ones(127, dtype=torch.bfloat16, device=cuda))
    refused("k_norm", k_norm=torch.ones(128, device=cuda))
    refused("k_cache must be on", k_cache=o["k_cache"])
    wide = torch.empty(4, 2, 16, 132, dtype=torch.bfloat16, device=cuda)
    refused("-2", k_cache=wide[..., :128], v_cache=wide[..., :128])
