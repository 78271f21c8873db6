"""Infinities in an adapter's B, and in h: both forms of lora_add give the definition's infinities and NaN, and keep the other
outputs within the bound of test_gpu_lora.py."""
import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, lora64
from gpu_util import note
from test_gpu_lora import call, operands

pytestmark = pytest.mark.gpu
INF = float("inf")


def check(o, out, splits):
    ref = lora64(o["y"], o["x"], o["A"], o["B"], o["ids"], o["scaling"], splits)
    out = out.cpu().double()
    assert ref.isinf().any() and torch.equal(out.isnan(), ref.isnan())
    assert torch.equal(out[ref.isinf()], ref[ref.isinf()])
    E = lora64(torch.zeros_like(o["y"]), o["x"].abs(), o["A"].abs(), o["B"].abs(), o["ids"], o["scaling"].abs(), splits)
    K, R = o["x"].shape[1], o["B"].shape[2]
    bound = ((K + R + 16) * F32_EPS + 2.0 ** -16) * E + F32_EPS * o["y"].double().abs() + BF16_HALF * ref.abs()
    fine = ref.isfinite()
    assert ((out - ref).abs()[fine] <= bound[fine]).all()


@pytest.mark.parametrize("rank", [8, 16, 40, 64, 136])     # the form for few rows of low ranks, and the other
def test_infinities_of_b(cuda, rank):
    """+inf and -inf against h of both signs; two of them in one output (NaN where their products differ in sign)."""
    for M, ids in ((1, [0]), (5, [0, 1, 0, -1, 1]), (20, [0] * 18 + [1, -1])):
        note(f"lora infinities of B rank={rank} M={M}")
        o = operands(M, 96, [50, 30], rank, 2, seed=rank + M, ids=ids)
        o["B"][0, 3, 0], o["B"][0, 60, rank - 1] = INF, -INF
        o["B"][0, 7, 1], o["B"][0, 7, 5] = INF, INF
        o["B"][1, 79, 2] = INF
        check(o, call(o, cuda, [50, 30]), [50, 30])


@pytest.mark.parametrize("rank", [8, 40])
def test_h_that_bf16_holds_exactly(cuda, rank):
    """h = +-1 and +-2^-20 exactly: nothing remains beyond its bf16 value, an infinity of B must meet no 0."""
    o = operands(4, 8, [16], rank, 1, ids=[0, 0, 0, 0])
    o["A"].zero_()
    o["A"][0, :, 0] = 1.0
    o["x"].zero_()
    o["x"][:, 0] = torch.tensor([1.0, -1.0, 2.0 ** -20, -2.0 ** -20])
    o["scaling"][:] = 1.0
    o["B"][0, 3, 2], o["B"][0, 5, 4] = INF, -INF
    check(o, call(o, cuda, None), [16])


@pytest.mark.parametrize("rank", [8, 40])
def test_an_infinite_h_meets_an_infinite_b(cuda, rank):
    o = operands(2, 8, [16], rank, 1, ids=[0, 0])
    o["A"][:], o["x"][0], o["x"][1], o["B"][:] = 1e30, 1e30, -1e30, 0.5
    o["B"][0, 4] = INF
    out = call(o, cuda, None).cpu().float()
    assert (out[0] == INF).all() and (out[1] == -INF).all()
