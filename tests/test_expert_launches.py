"""How many blocks a call of the experts' products may need: up to 2^22 of the format's largest, whichever blocks the pairs an expert
has on average would take. The CPU's part returns from the entry points and launches nothing (without a GPU a launch is an error of its
own); the GPU's runs calls that the blocks of their averages could not."""
import pytest
import torch

from conftest import gpu_available
from expert_util import make_experts, order64
from gpu_util import note
from test_expert_refusals import experts
from test_gpu_experts import check, ids_of, run

ABI = {"bf16": "bf16", "fp8": "fp8", "int4": "int4", "int4zp": "int4_zp"}
N = 1 << 25
COUNTS = {"bf16": 25, "fp8": 12, "int4": 12, "int4zp": 12}       # pairs of each of 12 experts: blocks of 32 (bf16) or 16
K = {"bf16": 8, "fp8": 16, "int4": 128, "int4zp": 128}


def contract(fmt, E, pairs, N):
    """Blocks as the header counts them."""
    side = 256 if fmt == "bf16" else 128
    return (pairs + min(pairs, E + 1) * (side - 1)) // side * -(-N // side)


@pytest.mark.skipif(gpu_available(), reason="addresses that are never read, as long as there is no GPU to launch on")
@pytest.mark.parametrize("fmt", list(ABI))
@pytest.mark.parametrize("gated", [0, 1])
def test_the_contract_is_what_is_refused(gemv_lib, fmt, gated):
    """Either side of the most blocks, at averages that every kind of blocks serves."""
    for E in (1, 8, 12, 64, 1024):
        for average in (1, 3, 12, 25, 40, 60, 100, 200, 400):
            pairs = E * average
            most = max(n for n in range(7, 26) if contract(fmt, E, pairs, 1 << n) <= 1 << 22)
            call = lambda n: experts(gemv_lib, fmt=ABI[fmt], E=E, pairs=pairs, rows=pairs, N=n, os=n, K=K[fmt],  # noqa: E731
                                     xs=K[fmt], gated=gated)
            assert call(1 << most) > 0, (E, average, most)
            if most < 25:
                assert contract(fmt, E, pairs, 2 << most) > 1 << 22 and call(2 << most) == -2, (E, average, most)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", list(ABI))
def test_larger_blocks_where_small_ones_are_too_many(cuda, fmt):
    """12 matrices of 2^25 rows: by blocks of 16 or 32 pairs 5.5 million, by the largest 1.8 to 3.7."""
    E, n = 12, COUNTS[fmt]
    small, _ = make_experts(fmt, E, 120, K[fmt], seed=3)
    columns = torch.cat([torch.arange(40), torch.arange(N // 2 - 20, N // 2 + 20), torch.arange(N - 40, N)]).to(cuda)
    raw = lambda t: t.view(torch.uint8) if t.element_size() == 1 else t  # noqa: E731
    W = [torch.zeros((E, N, *w.shape[2:]), dtype=raw(w).dtype, device=cuda) for w in small]
    for w, s in zip(W, small):
        w[:, columns] = raw(s).to(cuda)
    order, offsets = order64(ids_of([n] * E, n * E, 1), E)
    x = torch.randn(n * E, K[fmt], generator=torch.Generator().manual_seed(4)).bfloat16()
    note(f"experts of 2^25 rows {fmt}")
    out = run(fmt, W, None, x, order, offsets, cuda)
    check(out[:, columns], fmt, small, None, x, order, offsets, False)
    assert int(out.count_nonzero()) == int(out[:, columns].count_nonzero())
