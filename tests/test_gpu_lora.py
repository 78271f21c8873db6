"""ops.lora_add and GemvLib.lora_add against the definition in 64 bits.

Tolerance. With H = sum |A||x| of a value of h and E = scaling * sum |B| H over the rank: h is off by at most (K + 8) 2^-24 H
(fp32 sums), its two bf16 terms by 2^-16 of it, the second sum by (rank + 8) 2^-24, so
  |out - ref| <= ((K + rank + 16) 2^-24 + 2^-16) E + 2^-24 |y| + 2^-8 |ref|   (one rounding to bf16).
"""
import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, bits, lora64
from gpu_util import note
from paia_gemv import load_lib, ops

pytestmark = pytest.mark.gpu


def operands(M, K, splits, rank, adapters, seed=1, ids=None):
    g = torch.Generator().manual_seed(seed)
    N, S = sum(splits), len(splits)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    return {"y": r(M, N), "x": r(M, K), "A": (r(adapters, S * rank, K).float() * K ** -0.5).bfloat16(), "B": r(adapters, N, rank),
            "ids": torch.randint(-1, adapters, (M,), generator=g).int() if ids is None
            else torch.tensor(ids, dtype=torch.int32),
            "scaling": torch.rand(adapters, generator=g) + 0.5}


def call(o, dev, splits, **more):
    d = {k: (v if v is None else v.to(dev)) for k, v in o.items()}
    out = ops.lora_add(d["y"], d["x"], d["A"], d["B"], d["ids"], scaling=d["scaling"], splits=splits, **more)
    torch.cuda.synchronize()
    return out


def check(o, out, splits):
    ref = lora64(o["y"], o["x"], o["A"], o["B"], o["ids"], o["scaling"], splits)
    E = lora64(torch.zeros_like(o["y"]), o["x"].abs(), o["A"].abs(), o["B"].abs(), o["ids"], o["scaling"], splits)
    K, R = o["x"].shape[1], o["B"].shape[2]
    bound = ((K + R + 16) * F32_EPS + 2.0 ** -16) * E + F32_EPS * o["y"].double().abs() + BF16_HALF * ref.abs()
    worst = ((out.cpu().double() - ref).abs() - bound).max()
    assert worst <= 0, f"beyond the bound by {worst:.3e}"
    bare = (o["ids"] < 0) | (o["ids"] >= o["A"].shape[0])
    assert torch.equal(bits(out)[bare], bits(o["y"])[bare])


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 128, 136, 256])
@pytest.mark.parametrize("splits", [[64], [1003], [256, 40, 40], [7, 1, 300, 5], [512, 512]])
def test_ranks_and_slices(cuda, rank, splits):
    for M, K, adapters in ((1, 64, 1), (5, 3576, 3), (17, 1000, 2), (16, 8, 20)):
        note(f"lora M={M} K={K} splits={splits} rank={rank} adapters={adapters}")
        o = operands(M, K, splits, rank, adapters, seed=rank + M)
        check(o, call(o, cuda, splits), splits)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 600])
def test_row_counts(cuda, M):
    """Chunks of sixteen rows, launches of 256; every row its own adapter, all the same, two, and none."""
    for ids in (list(range(M)), [3] * M, [m % 2 for m in range(M)], [-1] * M, [m if m % 3 else -1 for m in range(M)]):
        for rank in (16, 40):
            note(f"lora M={M} rank={rank} ids={ids[:3]}..")
            o = operands(M, 264, [100], rank, max(M, 4), seed=M, ids=ids)
            check(o, call(o, cuda, None), [100])


def test_long_rows(cuda):
    o = operands(3, 18944, [3584], 64, 4, ids=[2, 0, 2])
    check(o, call(o, cuda, None), [3584])
    o = operands(16, 4096, [4096, 1024, 1024], 16, 16, ids=list(range(16)))
    check(o, call(o, cuda, [4096, 1024, 1024]), [4096, 1024, 1024])


def test_ids_outside_and_no_scaling(cuda):
    for rank in (8, 40):
        o = operands(6, 128, [96], rank, 3, ids=[-1, 3, 2 ** 31 - 1, -2 ** 31, 2, 0])
        o["scaling"] = None
        check(o, call(o, cuda, None), [96])


@pytest.mark.parametrize("rank", [24, 40])     # the form for few rows of low ranks, and the other
def test_in_place_strided_and_workspace(cuda, rank):
    """out = y in place, y, x and out as parts of wider tensors (even and odd offsets), a caller's workspace of NaN."""
    splits = [70, 58]
    o = operands(9, 256, splits, rank, 3)
    want = call(o, cuda, splits)
    d = {k: v.to(cuda) for k, v in o.items()}
    args = (d["x"], d["A"], d["B"], d["ids"])
    y = d["y"].clone()
    r = ops.lora_add(y, *args, scaling=d["scaling"], splits=splits, out=y)
    assert r is y and torch.equal(bits(y), bits(want))
    for left in (4, 3):
        wide = torch.full((9, 256), float("nan"), dtype=torch.bfloat16, device=cuda)
        part = wide[:, left:left + 128]
        part.copy_(d["y"])
        xw = torch.full((9, 512), float("nan"), dtype=torch.bfloat16, device=cuda)
        xw[:, 16:272] = d["x"]
        space = torch.full((load_lib().lora_add_workspace(9, 256, rank, splits) // 4,), float("nan"), device=cuda)
        ops.lora_add(part, xw[:, 16:272], *args[1:], scaling=d["scaling"], splits=splits, out=part, workspace=space)
        torch.cuda.synchronize()
        assert torch.equal(bits(part), bits(want)) and wide[:, :left].isnan().all() and wide[:, left + 128:].isnan().all()


@pytest.mark.parametrize("rank", [16, 40])
def test_not_finite_values_stay_in_their_rows(cuda, rank):
    """NaN and infinities in one row's x, in one adapter and in an adapter that nobody uses."""
    o = operands(20, 96, [80], rank, 4, ids=[0] * 10 + [1] * 10)
    want = call(o, cuda, None).cpu()
    o["A"][2], o["B"][3] = float("nan"), float("inf")
    o["x"][4, 7], o["x"][15, 0] = float("nan"), float("inf")
    got = call(o, cuda, None).cpu()
    assert got[4].isnan().all() and not got[15].isfinite().any()
    rows = [m for m in range(20) if m not in (4, 15)]
    assert torch.equal(bits(got[rows]), bits(want[rows]))


@pytest.mark.parametrize("rank", [8, 40])
def test_an_infinite_product_is_infinite(cuda, rank):
    """h beyond fp32's range: the remainder term must not turn the infinity into NaN."""
    o = operands(1, 8, [16], rank, 1, ids=[0])
    o["A"][:], o["x"][:], o["B"][:] = 1e30, 1e30, 0.5
    assert (call(o, cuda, None).cpu().float() == float("inf")).all()


def test_offsets_beyond_32_bits(cuda):
    """The last of adapters that fill 5 GiB of A and 5 of B, in both forms."""
    for R in (64, 16):
        far_adapters(cuda, 4096, 4096, R)


def far_adapters(cuda, K, N, R):
    L = 5 * 2 ** 30 // (R * K * 2)
    o = operands(3, K, [N], R, 2, ids=[1, 0, 1])
    want = call(o, cuda, None)
    A = torch.empty(L, R, K, dtype=torch.bfloat16, device=cuda)
    B = torch.empty(L, N, R, dtype=torch.bfloat16, device=cuda)
    A[L - 2:], B[L - 2:] = o["A"].to(cuda), o["B"].to(cuda)
    scaling = torch.ones(L, device=cuda)
    scaling[L - 2:] = o["scaling"].to(cuda)
    note("lora far adapters")
    got = ops.lora_add(o["y"].to(cuda), o["x"].to(cuda), A, B, (o["ids"] + (L - 2)).to(cuda), scaling=scaling)
    assert torch.equal(bits(got), bits(want))


@pytest.mark.parametrize("rank", [16, 40])
def test_graph_follows_the_ids(cuda, rank):
    """One captured call replayed with other requests in its rows, eager work between the replays."""
    splits = [200, 56]
    o = operands(8, 512, splits, rank, 5)
    d = {k: v.to(cuda) for k, v in o.items()}
    call_it = lambda: ops.lora_add(d["y"], d["x"], d["A"], d["B"], d["ids"], scaling=d["scaling"], splits=splits)  # noqa: E731
    call_it()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call_it()
    for ids in ([0] * 8, [-1] * 8, [4, 3, 2, 1, 0, 4, 3, 2], [1, -1, 1, -1, 1, 1, 1, 9]):
        d["ids"].copy_(torch.tensor(ids))
        junk = torch.randn(1 << 20, device=cuda).mul_(2.0)
        torch.cuda.synchronize()
        note(f"lora replay {ids}")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(call_it()))
        check({**o, "ids": torch.tensor(ids, dtype=torch.int32)}, out, splits)
        del junk


def test_c_abi_and_another_stream(cuda):
    splits = [96, 32]
    o = operands(7, 320, splits, 40, 3)
    want = call(o, cuda, splits)
    d = {k: v.to(cuda) for k, v in o.items()}
    lib, out = load_lib(), torch.empty(7, 128, dtype=torch.bfloat16, device=cuda)
    need = lib.lora_add_workspace(7, 320, 40, splits)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        space = torch.empty(need, dtype=torch.uint8, device=cuda)
        x = (d["x"].float() * 2.0).to(torch.bfloat16).div_(2.0)
        lib.lora_add(d["y"].data_ptr(), x.data_ptr(), d["A"].data_ptr(), d["B"].data_ptr(), d["ids"].data_ptr(),
                     d["scaling"].data_ptr(), out.data_ptr(), 7, 320, 40, splits, 3, space.data_ptr(), need)
    st.synchronize()
    assert torch.equal(bits(out), bits(want))


def test_no_rows(cuda):
    o = operands(2, 64, [32], 8, 2)
    d = {k: v.to(cuda) for k, v in o.items()}
    assert ops.lora_add(d["y"][:0], d["x"][:0], d["A"], d["B"], d["ids"][:0]).shape == (0, 32)


def test_refusals(cuda):
    o = operands(4, 64, [32], 8, 3)
    d = {k: v.to(cuda) for k, v in o.items()}

    def refused(match, splits=None, **change):
        a = {**d, "out": None, "workspace": None, **change}
        with pytest.raises(RuntimeError, match=match):
            ops.lora_add(a["y"], a["x"], a["A"], a["B"], a["ids"], scaling=a["scaling"], splits=splits, out=a["out"],
                         workspace=a["workspace"])

    refused("A must be", A=d["A"].float())
    refused("A must be", A=d["A"].transpose(1, 2).contiguous().transpose(1, 2))
    refused("B must be", B=d["B"][0])
    refused("same adapters", B=d["B"][:2].contiguous())
    refused("x must be", x=d["x"][:, :56])
    refused("x must be", x=d["x"].t().contiguous().t())
    refused("y must be", y=d["y"][:3])
    refused("out must be", out=torch.empty(4, 31, dtype=torch.bfloat16, device=cuda))
    refused("ids", ids=d["ids"].long())
    refused("ids must be on", ids=d["ids"].cpu())
    refused("scaling", scaling=torch.ones(2, device=cuda))
    refused("sum to N", splits=[16, 17])
    refused("rank rows", splits=[16, 16])
    refused("1 to 8", splits=[])
    w = {k: v.to(cuda) for k, v in operands(4, 64, [32], 40, 3).items()}
    refused("workspace", **w, workspace=torch.empty(8, device=cuda))
    refused("-2", A=d["A"][..., :60].contiguous(), x=d["x"][:, :60].contiguous())
    refused("-2", A=d["A"][:, :4].contiguous(), B=d["B"][..., :4].contiguous())
    refused("-2", splits=[32, 0], A=d["A"].repeat(1, 2, 1))
    odd = torch.empty(4, 68, dtype=torch.bfloat16, device=cuda)
    refused("-2", x=odd[:, 1:65])
