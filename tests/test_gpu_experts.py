"""ops.experts_bf16/fp8/int4/int4_zp and GemvLib's against the definition in 64 bits; tolerances as expert_util.experts64 derives
them. Row counts are chosen so that every form of the kernels runs: blocks of 16, 32, 64, 128 and 256 rows, and, where rows of
weights have 1024 bytes or more (DEEP), few rows an expert (up to 4, 8, 16 a block) whose K the waves of a block share."""
import pytest
import torch

from decode_util import bits
from expert_util import FORMATS, STEP, experts64, make_experts, order64
from gpu_util import note
from paia_gemv import load_lib, ops

pytestmark = pytest.mark.gpu

CALL = {"bf16": ops.experts_bf16, "fp8": ops.experts_fp8, "int4": ops.experts_int4, "int4zp": ops.experts_int4_zp}


DEEP = {"bf16": 512, "fp8": 1024, "int4": 2048, "int4zp": 2048}


def ids_of(counts, M, k, seed=0):
    """[M, k] ids with counts[e] pairs of expert e, the rest -1, in random places."""
    flat = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((M * k - sum(counts),), -1)])
    return flat[torch.randperm(M * k, generator=torch.Generator().manual_seed(seed))].view(M, k).int()


def run(fmt, W, bias, x, order, offsets, dev, gated=False, **more):
    if fmt != "int4":
        more["bias"] = None if bias is None else bias.to(dev)
    return CALL[fmt](*[w.to(dev) for w in W], x.to(dev), order.to(dev), offsets.to(dev), gated=gated, **more)


def check(out, fmt, W, bias, x, order, offsets, gated):
    want, bound = experts64(fmt, W, x, order, offsets, bias, gated)
    worst = ((out.cpu().double() - want).abs() - bound).max()
    assert worst <= 0, f"beyond the bound by {worst:.3e}"
    rest = order[int(offsets[-1]):].long()
    assert not bits(out)[rest].any()


def case(fmt, counts, N, K, k=1, gated=False, bias=False, shared=False, bare=0, seed=0, dev="cuda"):
    pairs = sum(counts) + bare
    M = -(-pairs // k)
    ids = ids_of(counts, M, k, seed)
    W, b = make_experts(fmt, len(counts), N, K, seed, bias and fmt != "int4")
    order, offsets = order64(ids, len(counts))
    x = torch.randn(M if shared else M * k, K, generator=torch.Generator().manual_seed(seed + 1)).bfloat16()
    note(f"experts {fmt} counts={counts[:6]} N={N} K={K} k={k} gated={gated} bias={bias} shared={shared} bare={bare}")
    out = run(fmt, W, b, x, order, offsets, dev, gated)
    torch.cuda.synchronize()
    check(out, fmt, W, b, x, order, offsets, gated)


COUNTS = {"single": [1], "few": [1, 0, 2, 0, 0, 1, 0, 0], "eight": [3, 1, 0, 5, 2, 8, 1, 4], "sixteen": [16, 3, 0, 17, 9, 1],
          "thirty": [33, 0, 31, 20], "sixty": [64, 65, 1, 50], "hundred": [129, 100, 0, 140], "many": [300, 257, 3],
          "more": [400, 310]}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("counts", list(COUNTS))
def test_row_counts(cuda, fmt, counts):
    for N, K, gated, bias in ((96, 384, False, True), (520, 256, True, False), (1003, 128, False, False), (258, 640, True, True)):
        case(fmt, COUNTS[counts], N, K, gated=gated, bias=bias, seed=len(counts))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 33, 255, 256, 257, 511, 514])
def test_columns(cuda, fmt, N):
    for counts, K in (([2, 1], 256), ([40, 30], 256), ([200, 150], 256), ([290, 200], 256), ([1, 1, 0], DEEP[fmt]), ([2, 5], DEEP[fmt])):
        case(fmt, counts, N, K, bias=True, seed=N)
        if N % 2 == 0:
            case(fmt, counts, N, K, gated=True, bias=True, seed=N)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tail", [0, 1, 2, 5, 9, 16])
def test_few_rows_share_k(cuda, fmt, tail):
    """Waves with and without whole stages, INT4 of odd and even numbers of groups, from one pair to 16 of an expert."""
    K = DEEP[fmt] + tail * STEP[fmt]
    for i, counts in enumerate(([1], [0, 4], [1, 0, 2, 0, 0, 1, 0, 0], [3, 1, 0, 5, 2, 0, 1], [9, 0, 0, 16, 1, 0, 8, 2], [5, 17, 1, 0])):
        case(fmt, counts, 70, K, k=1 + i % 3, gated=i % 2 == 0, bias=True, shared=True, bare=i % 4, seed=tail + i)


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_items_than_blocks(cuda, fmt):
    """Shares of several items, of several experts, of which some end within an expert."""
    case(fmt, [1, 2, 1, 0, 1, 2, 0, 1], 8000, DEEP[fmt], bias=True)
    case(fmt, [2] * 7, 4100, DEEP[fmt], gated=True)
    case(fmt, [1, 0, 1, 1] * 25, 514, DEEP[fmt], gated=True, bare=9)
    case(fmt, [5] * 8, 10300, 256, bias=True)          # blocks of 16, more than the chip holds at a time


@pytest.mark.parametrize("fmt", FORMATS)
def test_experts_of_many_chunks(cuda, fmt):
    """Groups of eight columns of blocks through six chunks and more, the last group narrower, other experts beside them."""
    case(fmt, [700, 30], 1300, 128, bias=True)
    case(fmt, [3, 0, 210, 0, 1, 0, 0, 2], 1300, 128, bare=3)
    case(fmt, [100, 7, 0, 0, 0, 0, 0, 0, 0, 0], 2050, 256, gated=True)


@pytest.mark.parametrize("fmt", ["int4", "int4zp"])
def test_infinite_scales(cuda, fmt):
    """A group whose scale is infinite, all of its values one above the zero point: infinite outputs, from whichever wave and whether
    the others have stages or none."""
    for K in (256, 1024, 2048, 2048 + 128, 4096):
        for counts in ([1, 1], [20, 3], [60, 50]):
            W, _ = make_experts(fmt, 2, 40, K)
            W = [w.clone() for w in W]
            ids = ids_of(counts, sum(counts), 1)
            order, offsets = order64(ids, 2)
            x = torch.rand(sum(counts), K, generator=torch.Generator().manual_seed(5)).bfloat16() + 0.5
            codes, group = W[0].view(torch.uint8), K // 128 - 1
            codes[:, 7, group * 64:group * 64 + 64] = 0x99
            W[1][:, 7, group] = float("inf")
            if fmt == "int4zp":
                W[2][:, 7, group // 2] = 0x88
            note(f"experts infinite scales {fmt} {K} {counts}")
            got = run(fmt, W, None, x, order, offsets, cuda).cpu()
            assert (got[:, 7] == float("inf")).all() and got[:, [i for i in range(40) if i != 7]].isfinite().all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_depths(cuda, fmt):
    """K from the least to longer than every wave's stages, with tails."""
    step = STEP[fmt]
    for K in (step, 2 * step, 3 * step, 64 + step, 128 + step, 512 + step, 1024, 1024 - step, 4096 + 128):
        K = -(-K // step) * step
        for counts in ([1], [9, 8], [48, 40], [130, 180], [300]):
            case(fmt, counts, 40, K, seed=K)


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_rows(cuda, fmt):
    """Rows beyond what a block keeps of INT4 metadata (K > 20480), and the longest projections' K."""
    for K in (18944, 24576):
        for counts in ([2, 1], [40, 3]):
            case(fmt, counts, 48, K, seed=K)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k", [1, 2, 8])
def test_shared_rows_and_bare_pairs(cuda, fmt, k):
    """A token's pairs share its row of x; pairs without an expert give zeros, all of them too."""
    for counts, bare in (([3, 0, 2, 4], 5), ([100, 60, 0, 90], 70), ([0, 0, 0, 0], 21), ([400, 300, 2], 11), ([0, 0, 0, 9], 0)):
        case(fmt, counts, 66, 256, k=k, shared=True, bare=bare, gated=True, seed=k)
    for counts, bare in (([0, 0, 0, 0], 3), ([0, 1, 0, 0], 2)):
        case(fmt, counts, 66, DEEP[fmt], k=k, shared=True, bare=bare, gated=True, seed=k)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("E", [63, 64, 65, 128, 200, 1024])
def test_many_experts(cuda, fmt, E):
    g = torch.Generator().manual_seed(E)
    counts = torch.randint(0, 4, (E,), generator=g)
    counts[torch.randint(0, E, (3,), generator=g)] = 37
    case(fmt, counts.tolist(), 18, 128, bare=6, seed=E)
    case(fmt, torch.randint(0, 2, (E,), generator=g).tolist(), 18, DEEP[fmt], bare=6, seed=E)


def poison(fmt, W, e):
    """Expert e's operands such that everything they touch is NaN (INT4: infinite or NaN scales)."""
    W = [w.clone() for w in W]
    if fmt == "fp8":
        W[0].view(torch.uint8)[e] = 0x7F
    else:
        W[0 if fmt == "bf16" else 1][e] = float("nan")
    return W


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,deep", [(2, False), (20, False), (50, False), (140, False), (300, False), (2, True), (7, True)])
def test_not_finite_values_stay_where_they_are(cuda, fmt, rows, deep):
    """Experts of NaN that nobody chose beside the ones in use, rows of NaN and infinities in x: the others keep their bits."""
    K = 3 * STEP[fmt] + (0 if "int4" in fmt else 64) + deep * DEEP[fmt]
    counts = [0, rows, 0, rows, 0]
    ids = ids_of(counts, 2 * rows, 1)
    order, offsets = order64(ids, 5)
    W, _ = make_experts(fmt, 5, 34, K)
    x = torch.randn(2 * rows, K, generator=torch.Generator().manual_seed(3)).bfloat16()
    note(f"experts not finite {fmt} {rows}")
    want = run(fmt, W, None, x, order, offsets, cuda).cpu()
    for e in (0, 2, 4):
        W = poison(fmt, W, e)
    x[0, 0], x[2, K - 1] = float("nan"), float("inf")
    got = run(fmt, W, None, x, order, offsets, cuda).cpu()
    assert got[0].isnan().all() and not got[2].isfinite().any()
    keep = [r for r in range(2 * rows) if r not in (0, 2)]
    assert torch.equal(bits(got[keep]), bits(want[keep]))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,deep", [(3, False), (30, False), (300, False), (1, True), (3, True)])
def test_strided_rows_and_what_lies_between(cuda, fmt, rows, deep):
    K, N = DEEP[fmt] if deep else 256, 37
    ids = ids_of([rows, rows], 2 * rows, 1)
    order, offsets = order64(ids, 2)
    W, b = make_experts(fmt, 2, N, K, bias=True)
    x = torch.randn(2 * rows, K, generator=torch.Generator().manual_seed(3)).bfloat16()
    note(f"experts strided {fmt} {rows}")
    want = run(fmt, W, b, x, order, offsets, cuda)
    xw = torch.full((2 * rows, K + 40), float("nan"), dtype=torch.bfloat16, device=cuda)
    xw[:, 8:8 + K] = x.to(cuda)
    for left in (3, 4):
        ow = torch.full((2 * rows, N + 9), float("nan"), dtype=torch.bfloat16, device=cuda)
        out = ow[:, left:left + N]
        run(fmt, W, b, xw[:, 8:8 + K], order, offsets, cuda, out=out)
        assert torch.equal(bits(out.contiguous()), bits(want))
        assert ow[:, :left].isnan().all() and ow[:, left + N:].isnan().all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_beyond_32_bits(cuda, fmt):
    """The first and last experts of 5 GiB of weights, in both kernels."""
    N, K = 8192, 8192
    E = 5 * 2 ** 30 // (N * {"bf16": 2 * K, "fp8": K}.get(fmt, K // 2))
    small, _ = make_experts(fmt, 2, N, K)
    W = [torch.zeros((E, *w.shape[1:]), dtype=torch.uint8 if w.element_size() == 1 else w.dtype, device=cuda) for w in small]
    for w, s in zip(W, small):
        w[0], w[E - 1] = s.view(w.dtype)[0].to(cuda), s.view(w.dtype)[1].to(cuda)
    columns = torch.cat([torch.arange(40), torch.arange(N - 40, N)])
    for pairs in (2, 13 * E):
        x = torch.randn(pairs, K, generator=torch.Generator().manual_seed(3)).bfloat16()
        ids = (torch.arange(pairs) % 2)[:, None]
        order, offsets = order64((ids * (E - 1)).int(), E)
        note(f"experts far {fmt} {E} {pairs}")
        view = [w.view(torch.float8_e4m3fn) if fmt == "fp8" and i == 0 else w for i, w in enumerate(W)]
        got = run(fmt, view, None, x, order, offsets, cuda)[:, columns.to(cuda)]
        check(got, fmt, [w.view(torch.uint8)[:, columns].view(w.dtype) if w.element_size() == 1 else w[:, columns]
                         for w in small], None, x, *order64(ids.int(), 2), False)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("E,K", [(3, 128), (40, 2048)])
def test_orders_that_are_not_in_order(cuda, fmt, E, K):
    """Offsets and pairs outside their ranges are not followed: what is right beside them is right, nothing else is written."""
    W, _ = make_experts(fmt, E, 33, K)
    x = torch.randn(40, K, generator=torch.Generator().manual_seed(3)).bfloat16()
    order, offsets = order64(ids_of([13, 13, 14] if E == 3 else [1] * 40, 40, 1), E)
    want = run(fmt, W, None, x, order, offsets, cuda)
    bad = order.clone()
    bad[5], bad[20], bad[39] = -1, 40, 2 ** 31 - 1
    out = torch.full((40, 33), 7.0, dtype=torch.bfloat16, device=cuda)
    note(f"experts bad order {fmt}")
    run(fmt, W, None, x, bad, offsets, cuda, out=out)
    lost = order[[5, 20, 39]].long()
    keep = [r for r in range(40) if r not in lost.tolist()]
    assert torch.equal(bits(out[keep]), bits(want[keep])) and (out[lost] == 7.0).all()
    for off in ([0, 1000, -5, 40], [40, 13, 26, 0], [-2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1]):
        note(f"experts bad offsets {fmt} {off}")
        run(fmt, W, None, x, order, torch.tensor(off + off[-1:] * (E - 3), dtype=torch.int32), cuda, out=out)
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,deep", [(6, False), (90, False), (2, True), (6, True)])
def test_graph_follows_the_order(cuda, fmt, M, deep):
    """One captured call replayed over other choices, eager work between the replays; every replay equals the eager call."""
    K = DEEP[fmt] if deep else 256
    W, _ = make_experts(fmt, 4, 130, K)
    d = [w.to(cuda) for w in W]
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(3)).bfloat16().to(cuda)
    order, offsets = (t.to(cuda) for t in order64(ids_of([M // 2] * 4, M, 2), 4))
    call = lambda: CALL[fmt](*d, x, order, offsets, gated=True)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for counts in ([2 * M, 0, 0, 0], [0, 0, 0, 0], [1, M, 0, M - 1], [M // 2] * 4):
        o, f = order64(ids_of(counts, M, 2, seed=counts[0]), 4)
        order.copy_(o), offsets.copy_(f)
        junk = torch.randn(1 << 20, device=cuda).mul_(2.0)
        torch.cuda.synchronize()
        note(f"experts replay {fmt} {counts}")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(call()))
        check(out, fmt, W, None, x.cpu(), o, f, True)
        del junk


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("E,K", [(3, 256), (20, 2048)])
def test_c_abi_and_another_stream(cuda, fmt, E, K):
    W, b = make_experts(fmt, E, 64, K, bias=fmt != "int4")
    x = torch.randn(10, K, generator=torch.Generator().manual_seed(3)).bfloat16()
    order, offsets = order64(ids_of([7, 8, 4] if E == 3 else [1] * 19, 10, 2), E)
    want = run(fmt, W, b, x, order, offsets, cuda)
    d, o, f = [w.to(cuda) for w in W], order.to(cuda), offsets.to(cuda)
    bd = None if b is None else b.to(cuda)
    lib, out = load_lib(), torch.empty_like(want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        xd = (x.to(cuda).float() * 2.0).bfloat16().div_(2.0)
        call = {"bf16": lib.experts_bf16, "fp8": lib.experts_fp8, "int4": lib.experts_int4, "int4zp": lib.experts_int4_zp}[fmt]
        more = {} if fmt == "int4" else {"bias_ptr": bd.data_ptr()}
        call(*[w.data_ptr() for w in d], xd.data_ptr(), 10, o.data_ptr(), f.data_ptr(), out.data_ptr(), E, 64, K, 20, **more)
    st.synchronize()
    assert torch.equal(bits(out), bits(want))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_of_x_beyond_2_gib(cuda, fmt):
    """Few rows that no 32-bit byte offset spans."""
    K = DEEP[fmt]
    W, _ = make_experts(fmt, 4, 50, K)
    x = torch.randn(2, K, generator=torch.Generator().manual_seed(3)).bfloat16()
    order, offsets = order64(torch.tensor([[3], [1]], dtype=torch.int32), 4)
    far = torch.empty(2 ** 30 + K + 8, dtype=torch.bfloat16, device=cuda).as_strided((2, K), (2 ** 30 + 8, 1))
    far.copy_(x)
    note(f"experts far rows {fmt}")
    out = CALL[fmt](*[w.to(cuda) for w in W], far, order.to(cuda), offsets.to(cuda))
    check(out, fmt, W, None, x, order, offsets, False)


def test_more_columns_than_shares(cuda):
    """One expert of 16 GiB, either side of the most columns that few rows take item by item."""
    N, K = 2 ** 24 + 64, 512
    W = torch.zeros(1, N, K, dtype=torch.bfloat16, device=cuda)
    x = torch.randn(1, K, generator=torch.Generator().manual_seed(3)).bfloat16()
    order, offsets = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    for n in (N - 65, N):
        some = torch.cat([torch.arange(50), torch.arange(n // 2 - 30, n // 2 + 30), torch.arange(n - 50, n)])
        w = torch.randn(1, len(some), K, generator=torch.Generator().manual_seed(n)).bfloat16()
        W[:, some.to(cuda)] = w.to(cuda)
        note(f"experts columns {n}")
        out = ops.experts_bf16(W[:, :n], x.to(cuda), order.to(cuda), offsets.to(cuda))
        check(out[:, some.to(cuda)], "bf16", (w,), None, x, order, offsets, False)
        some_zero = out.float().count_nonzero()
        assert some_zero <= len(some)
        W[:, some.to(cuda)] = 0


def test_int32_and_uint8_views(cuda):
    """INT4 codes as int32 words, e4m3 as bytes."""
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(3)).bfloat16()
    order, offsets = order64(ids_of([2, 2], 4, 1), 2)
    for fmt, view in (("int4", torch.int32), ("int4zp", torch.int32), ("fp8", torch.uint8)):
        W, _ = make_experts(fmt, 2, 32, 256)
        want = run(fmt, W, None, x, order, offsets, cuda)
        assert torch.equal(want, run(fmt, (W[0].view(view), *W[1:]), None, x, order, offsets, cuda))


@pytest.mark.parametrize("fmt", FORMATS)
def test_refusals(cuda, fmt):
    W, _ = make_experts(fmt, 3, 32, 256)
    x = torch.randn(4, 256).bfloat16()
    order, offsets = order64(ids_of([3, 3, 2], 4, 2), 3)
    base = dict(W=[w.to(cuda) for w in W], x=x.to(cuda), order=order.to(cuda), offsets=offsets.to(cuda), gated=False, out=None)

    def refused(match, **change):
        a = {**base, **change}
        with pytest.raises(RuntimeError, match=match):
            CALL[fmt](*a["W"], a["x"], a["order"], a["offsets"], gated=a["gated"], out=a["out"])

    w = base["W"]
    refused("W", W=[w[0][0], *w[1:]])
    refused("W", W=[w[0].float() if fmt in ("bf16",) else w[0].view(torch.int8), *w[1:]])
    refused("x must be", x=base["x"].float())
    refused("x must be", x=base["x"][:, :128])
    refused("x must be", x=base["x"].t().contiguous().t())
    refused("x must be on", x=x)
    refused("order", order=base["order"].long())
    refused("order", order=base["order"].view(4, 2))
    refused("offsets", offsets=base["offsets"][:3])
    refused("offsets must be on", offsets=offsets)
    refused("multiple of the rows", x=base["x"][:3].contiguous())
    refused("out must be", out=torch.empty(8, 31, dtype=torch.bfloat16, device=cuda))
    refused("out must be", gated=True, out=torch.empty(8, 32, dtype=torch.bfloat16, device=cuda))
    if len(w) > 1:
        refused("scale", W=[w[0], w[1][:2].contiguous(), *w[2:]])
        refused("scale", W=[w[0], w[1].double(), *w[2:]])
    if fmt == "int4zp":
        refused("zeros", W=[w[0], w[1], w[2][:, :1].contiguous()])
    wide = torch.empty(4, 260, dtype=torch.bfloat16, device=cuda)
    refused("-2", x=wide[:, 1:257])
    odd, _ = make_experts(fmt, 3, 33, 256)
    refused("even", W=[v.to(cuda) for v in odd], gated=True)
    assert CALL[fmt](*w, base["x"][:0], base["order"][:0], base["offsets"]).shape == (0, 32)
