"""Infinities in V that a token sees: the output is the definition's, infinite where one sign is seen and NaN where both are,
and the other dims keep the bounds of test_gpu_attention.py. Scores are moderate, so no weight of a position that is seen leaves
fp32's range and every product of a weight with an infinity is one."""
import math

import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, attention64
from gpu_util import note
from test_gpu_attention import call, operands

pytestmark = pytest.mark.gpu
INF = float("inf")


def plant(o, b, positions, dims=(1, 30, 62)):
    """+inf, -inf in a dim of V each, and NaN's two halves (+inf at the first position, -inf at the last) in a third."""
    page = o["v_cache"].shape[2]
    plus, minus, both = dims
    for i, p in enumerate(positions):
        row = o["v_cache"][int(o["table"][b, p // page]), :, p % page]
        row[:, plus], row[:, minus] = INF, -INF
        row[:, both] = INF if i == 0 else -INF


def check(o, out, lse, **more):
    ref, rlse, A, Q = attention64(o["q"], o["k_cache"], o["v_cache"], o["table"], o["lens"], **more)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert ref.isinf().any()
    assert torch.equal(out.isnan(), ref.isnan()), "NaN elsewhere than in the definition"
    assert torch.equal(out[ref.isinf()], ref[ref.isinf()]), "infinities elsewhere than in the definition"
    n, D = int(o["lens"].max()), o["q"].shape[-1]
    e, joins = (D + 16) * F32_EPS * Q, 2.0 ** -20 + (n / 32 + 64) * F32_EPS
    fine = ref.isfinite()
    bound = (2 * e[..., None] + joins + BF16_HALF) * A + BF16_HALF * ref.abs()
    assert ((out - ref).abs()[fine] <= bound[fine]).all()
    seen = rlse > -math.inf
    assert ((lse - rlse).abs() <= e + joins + 2.0 ** -22 * rlse.abs())[seen].all() and (lse[~seen] == -math.inf).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 7])
def test_one_token(cuda, dim, page):
    """One position alone (its weight is 1, nothing is left over), a few, a sequence of several pieces."""
    for lens, at in (([1], [0]), ([1, 2], [1]), ([40, 40], [0, 17, 39]), ([3001, 5], [0, 1500, 3000])):
        note(f"attention seen infinities dim={dim} page={page} lens={lens} at={at}")
        o = operands(lens, 1, 8, 2, dim, False, "hpd", page, seed=dim + page)
        plant(o, lens.index(max(lens)), at)
        check(o, *call(o, cuda))


@pytest.mark.parametrize("T,heads,window", [(3, 8, 0), (3, 8, 20), (5, 16, 0), (3, 40, 100)])
@pytest.mark.parametrize("dim", [64, 128])
def test_drafts(cuda, dim, T, heads, window):
    """Rows that all tokens see, that the last token alone sees and that has left a window; narrow tables and wide ones, whose
    blocks take several tiles of columns."""
    page, lens = 16, [333, 41]
    wide = -(-(300 << 20) // (2 * 2 * 2 * dim * 2 * page))
    for at in ([320, 325], [332], [331, 332], [333 - (T - 1) - max(window, 1), 330]):
        o = operands(lens, T, heads, 2, dim, False, "phd", page, seed=T + heads)
        plant(o, 0, at)
        note(f"attention seen infinities dim={dim} T={T} heads={heads} window={window} at={at}")
        check(o, *call(o, cuda, window=window), window=window)
        table = torch.full((2, wide), -1, dtype=torch.int32)
        table[:, :o["table"].shape[1]] = o["table"]
        got = call({**o, "table": table}, cuda, window=window)
        check(o, *got, window=window)
