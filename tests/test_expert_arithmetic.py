"""How the experts' blocks and waves find their work: the kernels' own arithmetic (csrc/expert_units.h) on the CPU, by the host's
compiler. For offsets in order every pair and tile is some block's exactly once and the launch has blocks enough; whatever the offsets
hold, what a block takes lies within the pairs."""
import ctypes
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

TESTS = Path(__file__).resolve().parent
CSRC = TESTS.parent / "paia-project_amd" / "csrc"
WAVES, CUS = 4, 256


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = tmp_path_factory.mktemp("units") / "expert_units_host.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(out),
                    str(TESTS / "expert_units_host.cpp")], check=True)
    lib = ctypes.CDLL(str(out))
    lib.host_most_chunks.restype = lib.host_most_blocks.restype = lib.host_most_items.restype = ctypes.c_int64
    lib.host_most_chunks.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    lib.host_share.restype, lib.host_share.argtypes = ctypes.c_uint64, [ctypes.c_uint64] * 3
    lib.host_share32.restype, lib.host_share32.argtypes = ctypes.c_uint32, [ctypes.c_uint32] * 3
    return lib


def units(host, offsets, R, E, BM, tiles):
    blocks = host.host_most_chunks(R, E, BM) * tiles
    o, out = np.array(offsets, dtype=np.int32), np.zeros((blocks, 5), dtype=np.int32)
    assert host.host_units(o.ctypes.data_as(ctypes.c_void_p), E, R, BM, tiles, blocks, out.ctypes.data_as(ctypes.c_void_p)) == 0
    return out[out[:, 0] >= 0]


def runs(host, offsets, R, E, MT, tiles, blocks):
    o, room = np.array(offsets, dtype=np.int32), 4 * (blocks + R + E) + 16
    out = np.zeros((room, 5), dtype=np.int32)
    n = host.host_runs(o.ctypes.data_as(ctypes.c_void_p), E, R, MT, tiles, blocks, room, out.ctypes.data_as(ctypes.c_void_p))
    assert n >= 0
    return out[:n]


def in_order(rng, E, R):
    cuts = sorted(rng.randint(0, R) for _ in range(E))
    if rng.random() < 0.5:
        cuts = sorted(rng.choice(cuts) for _ in range(E))
    return [0] + cuts


def of_any_kind(rng, E, R):
    return [rng.choice([rng.randint(-2 ** 31, 2 ** 31 - 1), rng.randint(-5, R + 5), 0, R]) for _ in range(E + 1)]


def sizes(rng):
    return (rng.choice([1, 2, 8, 63, 64, 65, 129, 200, 1024]), rng.choice([1, 2, 7, 64, 300, 1000, 5000]))


@pytest.mark.parametrize("seed", range(80))
def test_every_pair_and_tile_once(host, seed):
    rng = random.Random(seed)
    (E, R), BM, tiles = sizes(rng), rng.choice([16, 32, 64, 128, 256]), rng.choice([1, 3, 8, 9, 20])
    offsets = in_order(rng, E, R)
    seen = np.zeros((R, tiles), dtype=np.int64)
    for e, first, held, tile, chunks in units(host, offsets, R, E, BM, tiles):
        assert 0 < held <= BM and 0 <= tile < tiles
        if e == E:
            assert offsets[E] <= first and chunks == 0
        else:
            assert offsets[e] <= first and first + held <= offsets[e + 1] and chunks == -(-(offsets[e + 1] - offsets[e]) // BM)
        seen[first:first + held, tile] += 1
    assert (seen == 1).all()


@pytest.mark.parametrize("seed", range(80))
def test_few_rows_every_pair_and_tile_once(host, seed):
    """Items of pairs that have an expert; the blocks that are resident, or as many as there can be items."""
    rng = random.Random(seed)
    (E, R), MT, tiles = sizes(rng), rng.choice([4, 8, 16]), rng.choice([1, 3, 88, 896])
    offsets = in_order(rng, E, R)
    blocks = min(host.host_most_chunks(R, E, MT) * tiles, 3 * rng.choice([4, 80, CUS]))
    seen = np.zeros((R, tiles), dtype=np.int64)
    for e, first, held, tile, wide in runs(host, offsets, R, E, MT, tiles, blocks):
        assert 0 < held <= MT and wide > 0 and 0 <= tile and tile + wide <= tiles
        assert 0 <= e < E and offsets[e] <= first and first + held <= offsets[e + 1]
        seen[first:first + held, tile:tile + wide] += 1
    assert (seen[:offsets[E]] == 1).all() and not seen[offsets[E]:].any()


@pytest.mark.parametrize("seed", range(80))
def test_any_offsets_stay_within_the_pairs(host, seed):
    rng = random.Random(seed)
    (E, R), BM, tiles = sizes(rng), rng.choice([16, 64, 256]), rng.choice([1, 5])
    offsets = of_any_kind(rng, E, R)
    for e, first, held, tile, _ in units(host, offsets, R, E, BM, tiles):
        assert 0 <= e <= E and 0 <= tile < tiles and 0 < held <= BM and 0 <= first and first + held <= R, offsets
    for e, first, held, tile, wide in runs(host, offsets, R, E, 4, tiles, min(host.host_most_chunks(R, E, 4) * tiles, 768)):
        assert 0 <= e < E and 0 <= tile and tile + wide <= tiles and 0 < held <= 4 and 0 <= first and first + held <= R, offsets


@pytest.mark.parametrize("n", [1, 7, 8, 9, 100, 777])
def test_xcds_take_contiguous_ranges(host, n):
    places = [host.host_xcd(b, n) for b in range(n)]
    assert sorted(places) == list(range(n))
    for xcd in range(8):
        mine = places[xcd::8]
        assert mine == list(range(mine[0], mine[0] + len(mine))) if mine else True


@pytest.mark.parametrize("seed", range(40))
def test_waves_share_the_stages_of_a_row(host, seed):
    stages = random.Random(seed).randint(1, 300)
    begin = [host.host_wave_begin(stages, w, WAVES) for w in range(WAVES + 1)]
    assert begin[0] == 0 and begin[-1] == stages
    assert all(0 <= b - a <= -(-stages // WAVES) for a, b in zip(begin, begin[1:]))


@pytest.mark.parametrize("seed", range(40))
def test_shares_are_even(host, seed):
    """Of rows to clear, in 64 bits; of the most items in 32, whose bounds must not pass 32 bits for any number of blocks."""
    rng = random.Random(seed)
    n, blocks = rng.choice([0, 1, 255, 2 ** 20, 2 ** 42]), rng.choice([1, 7, 768, 1024])
    begin = [host.host_share(n, b, blocks) for b in range(blocks + 1)]
    assert begin[0] == 0 and begin[-1] == n and all(0 <= b - a <= -(-n // blocks) for a, b in zip(begin, begin[1:]))
    items = rng.randint(1, host.host_most_items())
    assert all(host.host_share32(items, b, blocks) == items * b // blocks for b in range(blocks + 1))


def test_what_a_launch_takes(host):
    """Grids stay below 2^32 threads; the most items by the most resident blocks below 2^32."""
    assert host.host_most_blocks() * 512 < 2 ** 32
    most = host.host_most_items()
    assert host.host_share32(most, 3 * CUS, 3 * CUS) == most and host.host_share32(most, 4095, 4095) == most


def splits(R, bins):
    if bins == 1:
        yield (R,)
        return
    for n in range(R + 1):
        for rest in splits(R - n, bins - 1):
            yield (n, *rest)


@pytest.mark.parametrize("E", [1, 2, 3])
def test_the_most_chunks_are_the_most(host, E):
    for R in range(1, 9):
        for BM in (2, 3, 4):
            assert host.host_most_chunks(R, E, BM) == max(sum(-(-n // BM) for n in s) for s in splits(R, E + 1))
