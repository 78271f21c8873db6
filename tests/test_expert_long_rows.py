"""The experts' products at the longest K, bit for bit. Weights, scales and x are small integers and powers of two, so that every sum
of the formats' kernels is exact in fp32, in whatever order and with INT4's zero points taken apart: |terms| add up to less than 2^22
(at most 15 * 4 * 2 a column, 24704 columns), in whole units. What is left is the output's rounding, the same in the kernels and here.
The CPU's part plants the mistake that the GPU's is there to find, in the expected values: a few columns left out."""
import pytest
import torch

from expert_util import FORMATS, STEP, order64, weights64
from gpu_util import note
from test_gpu_experts import ids_of, run

E, N = 2, 48
DEPTHS = (18944, 24576, "24576 and a step")
# from one pair an expert to blocks of 256, every form of every format among them
COUNTS = ([1, 1], [2, 1], [6, 4], [14, 16], [25, 24], [20, 30], [40, 44], [60, 50], [100, 60], [120, 130], [300, 200])


def depth(fmt, K):
    return 24576 + STEP[fmt] if isinstance(K, str) else K


def operands(fmt, K, gated, seed):
    """(weights, bias or None). The first N rows of a gated matrix are gates of 2 * (16 or 7 * 4), whatever else x holds: such a gate
    is its own silu in fp32."""
    g = torch.Generator().manual_seed(seed)
    rows = 2 * N if gated else N
    b = torch.randint(-50, 51, (E, rows), generator=g).bfloat16()
    b[:, :N] *= 0 if gated else 1
    if fmt in ("bf16", "fp8"):
        W = torch.randint(-4, 5, (E, rows, K), generator=g)
        if gated:
            W[:, :N] = 0
            W[:, :N, 0] = 16
        if fmt == "bf16":
            return (W.bfloat16(),), b
        s = torch.randint(-2, 3, (E, rows), generator=g).float().exp2()
        if gated:
            s[:, :N] = 1.0
        return (W.float().to(torch.float8_e4m3fn), s), b
    q = torch.randint(0, 16, (E, rows, K), generator=g)
    s = torch.randint(0, 3, (E, rows, K // 128), generator=g).float().exp2()
    z = torch.randint(0, 256, (E, rows, (K // 128 + 1) // 2), dtype=torch.uint8, generator=g)
    if gated:
        q[:, :N] = 8
        q[:, :N, 0] = 15
        s[:, :N, 0] = 4.0
        z[:, :N] = 0x88
    W = (q[..., ::2] | q[..., 1::2] << 4).to(torch.uint8)
    return ((W, s.half()), None) if fmt == "int4" else ((W, s.bfloat16(), z), b)


def rows_of(pairs, K, seed):
    x = torch.randint(-2, 3, (pairs, K), generator=torch.Generator().manual_seed(seed)).bfloat16()
    x[:, 0] = 2.0
    return x


def expected(fmt, W, bias, x, order, offsets, gated, lost=slice(0, 0)):
    """The definition, exact in 64 bits, rounded once; without the columns `lost` of the values."""
    out = torch.empty(len(order), N, dtype=torch.bfloat16)
    for e in range(E):
        p = order[int(offsets[e]):int(offsets[e + 1])].long()
        w = weights64(fmt, W, e)[0]
        w[-N:, lost] = 0.0
        y = x[p].double() @ w.t()
        assert (x[p].double().abs() @ w.abs().t()).max() < 2 ** 22
        if bias is not None:
            y = y + bias[e].double()
        if gated:
            assert (y[:, :N] >= 32).all()
            y = y[:, :N] * y[:, N:]
        out[p] = y.float().bfloat16()
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gated", [False, True])
def test_lost_columns_show(fmt, gated):
    """The fewest pairs, and one step of columns (INT4: half a group) left out at the start, in the middle and at the end."""
    for i, K in enumerate(DEPTHS):
        K, step = depth(fmt, K), min(STEP[fmt], 64)
        W, b = operands(fmt, K, gated, i)
        order, offsets = order64(ids_of([1, 1], 2, 1), E)
        x = rows_of(2, K, i)
        right = expected(fmt, W, b, x, order, offsets, gated)
        for at in (step, K // 2 // step * step, K - step):
            wrong = expected(fmt, W, b, x, order, offsets, gated, slice(at, at + step))
            assert (wrong != right).float().mean() > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", DEPTHS)
@pytest.mark.parametrize("gated", [False, True])
def test_long_rows_are_exact(cuda, fmt, K, gated):
    K = depth(fmt, K)
    W, b = operands(fmt, K, gated, 1)
    for i, counts in enumerate(COUNTS):
        order, offsets = order64(ids_of(counts, sum(counts), 1, i), E)
        x = rows_of(sum(counts), K, i)
        note(f"experts of long rows {fmt} K={K} {counts} gated={gated}")
        out = run(fmt, W, b, x, order, offsets, cuda, gated).cpu()
        assert torch.equal(out, expected(fmt, W, b, x, order, offsets, gated)), counts
