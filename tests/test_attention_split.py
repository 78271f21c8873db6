"""How paged attention splits sequences into pieces, replayed on the CPU: the kernels derive the split from lengths that only
the device knows, within a grid and a workspace that the host fixed before (csrc/paged_attention.hip: piece_tiles, pieces_of,
attention_plan). Every tile must lie in exactly one piece and the pieces must fit the grid, whatever the lengths are."""
import random

import pytest

TILE, MIN_TILES, WAVES = 32, 8, 4


def span(n, T, window, max_len):
    n = min(max(n, 0), max_len)
    tile0 = max(0, n - (T - 1) - window) // TILE if window else 0
    return tile0, -(-n // TILE) - tile0


def pieces_of(tiles, most):
    n = max(1, -(-tiles // most))
    each = max(1, -(-tiles // n))
    return max(1, -(-tiles // each)), each


def piece_tiles(total, B, target):
    aim = max(target - B, (target + 1) // 2)
    return -(-max(-(-total // aim), MIN_TILES) // WAVES) * WAVES


def items_bound(B, target, max_len):
    per_seq = (max_len // TILE + 1 + MIN_TILES - 1) // MIN_TILES
    return min(max(target, (target + 1) // 2 + B), per_seq * B)


@pytest.mark.parametrize("seed", range(40))
def test_pieces_cover_every_tile_once_and_fit(seed):
    r = random.Random(seed)
    for _ in range(60):
        B, target, T = r.choice([1, 2, 3, 16, 63, 64, 65, 200]), r.choice([1, 2, 7, 64, 96, 128, 768]), r.choice([1, 2, 5])
        max_len = r.choice([0, 1, 31, 32, 256, 257, 5000, 131072, 2 ** 31 - 5000])
        window = r.choice([0, 0, 1, 33, 4096])
        lens = [r.choice([0, 1, max_len, r.randint(0, max(1, max_len)), r.randint(0, 2 ** 31 - 1)]) for _ in range(B)]
        spans = [span(n, T, window, max_len) for n in lens]
        most = piece_tiles(sum(t for _, t in spans), B, target)
        used = 0
        for tile0, tiles in spans:
            n, each = pieces_of(tiles, most)
            used += n
            assert each <= most or tiles <= most
            ends = [(min(tiles, j * each), min(tiles, (j + 1) * each)) for j in range(n)]
            assert ends[0][0] == 0 and ends[-1][1] == tiles
            assert all(a[1] == b[0] for a, b in zip(ends, ends[1:]))
            assert all(a < b for a, b in ends) or tiles == 0
            assert tile0 >= 0 and tiles >= 0
        assert used <= items_bound(B, target, max_len) or max_len == 0, (used, B, target, max_len)
        if (max_len // TILE + 1 + MIN_TILES - 1) // MIN_TILES <= 1:
            assert used == B


def test_uniform_lengths_use_what_is_aimed_at():
    """Equal sequences: between half and all of the pieces aimed at, and never more."""
    for B in (1, 4, 16):
        for n in (4096, 32768, 131072):
            most = piece_tiles(B * (n // TILE), B, 64)
            used = B * pieces_of(n // TILE, most)[0]
            assert 32 <= used <= 64 or most == MIN_TILES
