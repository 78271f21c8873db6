"""ops.route_experts and ops.expert_order against the definition in 64 bits: choices and order are equal, a weight is off by its
rounding to fp32 and what 64-bit arithmetic leaves (k + 300 roundings of 2^-53 at most, below 2^-43)."""
import math

import pytest
import torch

from expert_util import order64, route64
from gpu_util import note
from paia_gemv import load_lib, ops

pytestmark = pytest.mark.gpu


def check(logits, k, got, bias=None, **more):
    ids, weights, order, offsets = (t.cpu() for t in got)
    want_ids, want_w = route64(logits.cpu(), k, None if bias is None else bias.cpu(), **more)
    assert torch.equal(ids, want_ids)
    assert ((weights.double() - want_w).abs() <= (2.0 ** -24 + 2.0 ** -43) * want_w.abs() + 2.0 ** -150).all()
    want_order, want_offsets = order64(want_ids, logits.shape[1])
    assert torch.equal(order, want_order) and torch.equal(offsets, want_offsets)


def random_logits(M, E, dtype, seed=0, dev="cuda"):
    return torch.randn(M, E, generator=torch.Generator().manual_seed(seed + M + E)).mul_(2.0).to(dtype).to(dev)


@pytest.mark.parametrize("E", [1, 2, 7, 60, 64, 65, 128, 160, 256, 257, 512, 1000, 1023, 1024])
@pytest.mark.parametrize("M", [1, 31, 32, 33, 64, 200])
def test_sizes(cuda, E, M):
    for dtype in (torch.bfloat16, torch.float32):
        for k in {1, min(E, 4), min(E, 8), min(E, 64)}:
            for scoring, renormalize in (("softmax", True), ("sigmoid", True), ("softmax", False)):
                if k == 64 and M > 40 or (scoring == "sigmoid") != (dtype == torch.float32) and M == 200:
                    continue
                note(f"route M={M} E={E} k={k} {dtype} {scoring} {renormalize}")
                x = random_logits(M, E, dtype)
                more = dict(scoring=scoring, renormalize=renormalize, scale=1.0 if renormalize else 2.5)
                bias = torch.randn(E, generator=torch.Generator().manual_seed(E)).mul_(0.1).to(cuda) if scoring == "sigmoid" else None
                check(x, k, ops.route_experts(x, k, bias=bias, **more), bias, **more)


@pytest.mark.parametrize("M", [255, 256, 257, 4095, 4097, 20000])
def test_many_tokens(cuda, M):
    for E, k in ((16, 2), (256, 8)):
        note(f"route M={M} E={E} k={k}")
        x = random_logits(M, E, torch.float32)
        got = ops.route_experts(x, k)
        want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k].int()
        assert torch.equal(got[0], want)
        order, offsets = order64(want.cpu(), E)
        assert torch.equal(got[2].cpu(), order) and torch.equal(got[3].cpu(), offsets)
        check(x[:50], k, ops.route_experts(x[:50], k))
        x = x.bfloat16()                                 # ties in many rows
        got = ops.route_experts(x, k)
        assert torch.equal(got[0], torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k].int())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lower_index(cuda, dtype):
    for E in (64, 200, 1024):
        x = torch.zeros(5, E, device=cuda, dtype=dtype)
        x[1, ::2] = -0.0
        x[2, 3::5] = 1.0
        x[3] = torch.arange(E, device=cuda) % 3
        x[4] = -7.0
        x[4, 1::3] = -7.03125
        for scoring in ("softmax", "sigmoid"):
            note(f"route ties E={E} {scoring}")
            check(x, 8, ops.route_experts(x, 8, scoring=scoring), scoring=scoring)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_closed_experts(cuda, scoring):
    """-inf, NaN and the types' lowest values; rows with fewer open experts than k, and with none."""
    for dtype in (torch.bfloat16, torch.float32):
        x = random_logits(9, 40, dtype)
        x[0, 3:] = -math.inf
        x[1] = -math.inf
        x[2, 5], x[2, 17:30] = math.nan, -math.inf
        x[3] = math.nan
        x[4] = torch.finfo(dtype).min
        x[5, 2:] = torch.finfo(dtype).min
        x[6, 0] = torch.finfo(dtype).max
        x[7] = -1e4
        bias = torch.zeros(40, device=cuda)
        if scoring == "sigmoid":
            bias[7], bias[8], bias[9], bias[11] = -math.inf, math.nan, 1e30, math.inf
        note(f"route closed {dtype} {scoring}")
        b = bias if scoring == "sigmoid" else None
        for renormalize in (True, False):
            check(x, 6, ops.route_experts(x, 6, bias=b, scoring=scoring, renormalize=renormalize), b, scoring=scoring,
                  renormalize=renormalize)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_logits(cuda, dtype):
    """An infinite logit is chosen first; its softmax is NaN, as inf - inf is."""
    x = random_logits(2, 64, dtype)
    x[0, 9] = math.inf
    note("route infinite")
    ids, w, _, _ = ops.route_experts(x, 4)
    assert int(ids[0, 0]) == 9 and w[0].isnan().all() and w[1].isfinite().all()
    ids, w, _, _ = ops.route_experts(x, 4, scoring="sigmoid", renormalize=False)
    assert int(ids[0, 0]) == 9 and float(w[0, 0]) == 1.0


def test_order_of_given_ids(cuda):
    """Ids outside the experts, the same expert twice, one expert for all, none; both launches."""
    g = torch.Generator().manual_seed(5)
    for M in (1, 20, 500):
        for E in (5, 64, 1024):
            for ids in (torch.randint(-2, E + 2, (M, 6), generator=g), torch.zeros(M, 6), torch.full((M, 6), -1),
                        torch.full((M, 6), E - 1), torch.full((M, 6), 2 ** 31 - 1)):
                note(f"expert_order M={M} E={E} {ids[0, :2].tolist()}")
                ids = ids.int()
                order, offsets = ops.expert_order(ids.to(cuda), E)
                want = order64(ids, E)
                assert torch.equal(order.cpu(), want[0]) and torch.equal(offsets.cpu(), want[1])


def test_strides_workspace_and_streams(cuda):
    wide = random_logits(100, 200, torch.bfloat16)
    x = wide[:, 40:137]
    want = ops.route_experts(x.contiguous(), 5)
    lib = load_lib()
    need = lib.route_experts_workspace(100, 97, 5)
    assert need == ops.route_experts_workspace(100, 97, 5) > 0 and ops.route_experts_workspace(32, 97, 5) == 0
    space = torch.full((need,), 255, dtype=torch.uint8, device=cuda)
    note("route strided, a workspace")
    for a, b in zip(ops.route_experts(x, 5, workspace=space), want):
        assert torch.equal(a, b)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        made = [torch.empty_like(t) for t in want]
        lib.route_experts(x.data_ptr(), *[t.data_ptr() for t in made], 100, 97, 5, space.data_ptr(), need, logits_stride=200)
        lib.expert_order(made[0].data_ptr(), made[2].data_ptr(), made[3].data_ptr(), 100, 97, 5, space.data_ptr(), need)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(made, want))


@pytest.mark.parametrize("M", [7, 300])
def test_graph_follows_the_logits(cuda, M):
    x = random_logits(M, 64, torch.float32)
    ops.route_experts(x, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.route_experts(x, 4)
    for seed in (1, 2, 3):
        x.copy_(random_logits(M, 64, torch.float32, seed=seed))
        if seed == 2:
            x[M // 2:] = -math.inf
        torch.cuda.synchronize()
        note(f"route replay {seed}")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ops.route_experts(x, 4)))
        check(x, 4, got)


def test_no_tokens_and_refusals(cuda):
    x = random_logits(6, 16, torch.float32)
    ids, w, order, offsets = ops.route_experts(x[:0], 3)
    assert ids.shape == (0, 3) and w.shape == (0, 3) and order.numel() == 0 and offsets.tolist() == [0] * 17
    assert ops.expert_order(ids, 16)[1].tolist() == [0] * 17

    def refused(match, logits=x, k=3, **more):
        with pytest.raises(RuntimeError, match=match):
            ops.route_experts(logits, k, **more)

    refused("logits must be", logits=x.double())
    refused("logits must be", logits=x.t())
    refused("k must be", k=17)
    refused("k must be", k=0)
    refused("scoring", scoring="tanh")
    refused("bias goes with", bias=torch.zeros(16, device=cuda))
    refused("bias must be", bias=torch.zeros(15, device=cuda), scoring="sigmoid")
    refused("bias must be on", bias=torch.zeros(16), scoring="sigmoid")
    refused("workspace", logits=random_logits(100, 16, torch.float32), workspace=torch.empty(8, device=cuda))
    refused("-2", logits=random_logits(2, 1025, torch.float32))
    refused("-2", logits=random_logits(2, 128, torch.float32), k=65)
    for bad in (ids.long(), ids[0:0, 0], torch.zeros(4, 4, dtype=torch.int32, device=cuda).t()[:, :2]):
        with pytest.raises(RuntimeError, match="ids must be"):
            ops.expert_order(bad, 16)
    with pytest.raises(RuntimeError, match="-2"):
        ops.expert_order(torch.zeros(2, 2, dtype=torch.int32, device=cuda), 1025)
